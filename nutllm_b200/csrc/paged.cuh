#pragma once
/* Device helpers of the paged KV cache operators (paged_*.cu). */
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "common.cuh"
#include "kernels.h"
#include "paged.h"

namespace nut {

/* The paged kernels are set up while the kernel before them in the stream
 * drains: what that one wrote may be read, and its buffers written, after
 * begin_kernel().  (None lets the next one in earlier than its own last
 * block: waiting blocks of the attention would crowd the kernel they wait for,
 * 97 against 82 us for a sparse step of 32 sequences.) */
__device__ __forceinline__ void begin_kernel() { asm volatile("griddepcontrol.wait;\n" ::: "memory"); }

template <typename... Params, typename... Args>
cudaError_t launch_kernel(void (*kernel)(Params...), dim3 grid, int threads, size_t bytes, cudaStream_t stream,
                          int cluster, Args... args) {
    cudaLaunchConfig_t config{};
    config.gridDim = grid;
    config.blockDim = dim3(threads);
    config.dynamicSmemBytes = bytes;
    config.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    config.attrs = attr;
    config.numAttrs = cluster > 1 ? 2 : 1;
    count_launches(1);
    return cudaLaunchKernelEx(&config, kernel, args...);
}

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

/* Rounds to nearest; fp16 saturates at +-65504 and keeps NaN. */
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) {
    return __float2half_rn(v > 65504.0f ? 65504.0f : v < -65504.0f ? -65504.0f : v);
}
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) {
    return __float2bfloat16_rn(v);
}

__device__ __forceinline__ void paged_fail(const PagedPool &p, int bit) { atomicOr(p.error, bit); }

/* Slots in use of sequence s; 0, with the error recorded, when the length
 * is not one the table can hold. */
__device__ __forceinline__ int checked_length(const PagedPool &p, int length) {
    if (length < 0 || length > p.capacity) {
        paged_fail(p, kPagedBadLength);
        return 0;
    }
    return length;
}

/* Page number of logical page j of sequence s, or -1. */
__device__ __forceinline__ int lookup(const PagedPool &p, int s, int j) {
    const int page = p.table[int64_t(s) * p.max_pages + j];
    return unsigned(page) < unsigned(p.n_pages) ? page : -1;
}

/* Page number of logical page j of sequence s, or -1 (recorded). */
__device__ __forceinline__ int checked_page(const PagedPool &p, int s, int j) {
    const int page = p.table[int64_t(s) * p.max_pages + j];
    if (unsigned(page) >= unsigned(p.n_pages)) {
        paged_fail(p, kPagedBadPage);
        return -1;
    }
    return page;
}

/* Sequence of attention row r and the slots it sees (0 for a bad row). */
__device__ __forceinline__ int row_span(const PagedPool &p, const int32_t *row_sequence,
                                        const int32_t *row_length, int r, int &length) {
    int s = row_sequence ? row_sequence[r] : r;
    if (unsigned(s) >= unsigned(p.sequences)) {
        paged_fail(p, kPagedBadSequence);
        length = 0;
        return 0;
    }
    length = checked_length(p, row_length ? row_length[r] : p.lengths[s]);
    return s;
}

/* Power of two u, at least 2^-126, least with top <= 127 u (0 for top = 0):
 * top = m 2^e with 1 <= m < 2 needs u = 2^(e - 6), or twice that when
 * m > 127 / 64. */
__device__ __forceinline__ float unit_of(float top) {
    if (!(top > 0.0f))
        return 0.0f;
    const uint32_t b = __float_as_uint(top);
    int e = int(b >> 23) - 127 - 6;
    if ((b & 0x7fffffu) > 0x7e0000u) /* mantissa of 127 / 64 */
        e++;
    if (e < -126)
        e = -126;
    return __uint_as_float(uint32_t(e + 127) << 23);
}

/* NaN counts as 0, infinities as the largest finite float. */
__device__ __forceinline__ float finite_key(float v) {
    return v != v ? 0.0f : fminf(fmaxf(v, -3.402823466e38f), 3.402823466e38f);
}

} // namespace nut
