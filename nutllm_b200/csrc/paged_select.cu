/* Choosing pages by their key bounds (nut_paged_select).
 *
 * score(page) = max_g u_g U sum_d max(x_gd M_d, x_gd L_d), with x the query
 * head in 8 bits, M and L the page's greatest and least key in 8 bits, u and
 * U powers of two.  As max(x M, x L) = max(x, 0) M + min(x, 0) L, the sum is
 * one product of [M | L] with [max(x, 0) | min(x, 0)]: mma.sync m16n8k32 in
 * 8 bits, 16 pages by 8 query heads (of one row, or of two or four).  The sum is at most
 * 256 * 127 * 128 < 2^24 in size, so it is exact in an int and in fp32,
 * whatever its order; what the units carry beyond fp32's range counts as its
 * greatest number.
 *
 * It reads 2 head_dim + 4 bytes of each page and kv head, a 32nd of what the
 * page's 16 keys and values take in 16 bits.  35 MB of them (32 sequences of
 * up to 1,024 pages, 8 heads of 128) take 15 us, bound by the look-ups that
 * precede them (length, table, bounds) and the blocks' barriers, and choosing
 * 64 of each 6 us more.  256 rows of one prompt choosing 64 of 512 pages
 * take 32 us: 11 of them the choice, a warp for each row's.
 */
#include <cstdint>
#include <cuda_runtime.h>

#include "paged.cuh"
#include "paged_choose.cuh"
#include "stream.cuh"

namespace nut {
namespace {

constexpr int kWarps = 8;
constexpr int kPages = 16;  /* of a warp's product */
constexpr int kHeads = 8;   /* columns of a warp's product */
constexpr int kMostRows = 8; /* of a block, where rows can share a sequence */
constexpr float kMostFloat = 3.402823466e38f;
/* Most pages of a row that its block chooses from at once, in shared memory
 * and 16 registers a lane.  A table of 512 and of 513 pages, which the forms
 * below take in a second launch: 32 sequences 15.9 against 13.4 + 5.9 us, 256
 * prompt rows 26.7 against 26.2 + 13.4 (bounds out of L2).  1,024 against 1,025
 * pages, from registers and from histograms: 14.4 + 5.7 against 15.1 + 8.1. */
constexpr int kFusedPages = 512;

/* A warp writes the `n` first-ranked of a row's `pages` scores (at most 32 N,
 * in shared memory) to out, ascending, -1 behind.  Lanes own every 32nd
 * page, so that reads meet no bank twice and a ballot ranks a whole step
 * (scores and choice for 256 prompt rows of 512 pages, 8 kv heads: 41.8 us;
 * with 16 neighbouring pages a lane 42.8). */
template <int N>
__device__ __forceinline__ void choose_in_warp(const float *score, int pages, int n, int32_t *out) {
    const int lane = threadIdx.x & 31, want = min(n, pages);
    uint32_t k[N], threshold = 0;
#pragma unroll
    for (int e = 0; e < N; e++)
        k[e] = e * 32 + lane < pages ? ordered_bits(score[e * 32 + lane]) : 0u;
    int quota = want;
    if (want < pages) {
        WarpSums sum;
        search_largest(k, want, sum, threshold, quota);
    }
    const uint32_t before = (1u << lane) - 1u;
    int ties = 0, to = 0;
#pragma unroll
    for (int e = 0; e < N; e++) {
        const bool there = e * 32 + lane < pages, tie = there && k[e] == threshold;
        const uint32_t tied = __ballot_sync(0xffffffffu, tie);
        const bool chosen = (there && k[e] > threshold) || (tie && ties + __popc(tied & before) < quota);
        const uint32_t all = __ballot_sync(0xffffffffu, chosen);
        if (chosen)
            out[to + __popc(all & before)] = e * 32 + lane;
        ties += __popc(tied);
        to += __popc(all);
    }
    for (int i = want + lane; i < n; i += 32)
        out[i] = -1;
}

/* log2 of a product's columns for each row: groups of up to four heads leave room
 * for the heads of two or four rows (512 pages, 256 prompt rows of 8 x 4
 * heads: 34.0 against 41.8 us). */
__host__ __device__ constexpr int columns_of(int group) { return group > 4 ? 3 : group > 2 ? 2 : 1; }

/* Scores of 16 pages at a time for the rows of a block, KC 64-byte pieces
 * of bounds a page.  A lane loads 16 neighbouring bytes of two pages for two
 * products: which 32 of the 64 bytes meet in one product does not matter as
 * long as both operands take the same ones.  The first pages' bounds are on
 * their way (three look-ups one after another) while the queries are put
 * into 8 bits.  kFused: the block has all of its rows' pages, keeps the
 * scores in shared memory and chooses, a warp for each row. */
template <typename R, int KC, bool kFused>
__global__ void __launch_bounds__(kWarps * 32, KC <= 4 ? 3 : 2)
    score_kernel(const __grid_constant__ PagedSelect a, int rows_each, int pages_each) {
    constexpr int kWidth = KC * 64, kPitch = kWidth + 64; /* pitch: rows in different banks */
    constexpr int kBatch = 4;                             /* heads of a warp that load together */
    extern __shared__ __align__(16) int8_t queries[];     /* [columns][kPitch], kFused: then the scores */
    __shared__ float units[kMostRows * kHeads];
    __shared__ int sequence_of[kMostRows], pages_of[kMostRows], limit_of[kMostRows];
    __shared__ int run_end[kMostRows], run_pages[kMostRows];
    const PagedPool &p = a.p;
    const int head = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int g = lane >> 2, t = lane & 3, D = p.head_dim;
    const int row0 = int(blockIdx.z) * rows_each, rows = min(rows_each, a.rows - row0);
    const int j_from = int(blockIdx.x) * pages_each, j_to = j_from + pages_each;
    const int shift = columns_of(p.group), span = 1 << shift, together = kHeads >> shift; /* columns of a row; rows of a product */
    float *kept = reinterpret_cast<float *>(queries + max(rows_each * span, kHeads) * kPitch); /* [rows_each][kFusedPages] */
    begin_kernel();
    if (int(threadIdx.x) < rows) {
        int length;
        sequence_of[threadIdx.x] = row_span(p, a.row_sequence, a.row_length, row0 + int(threadIdx.x), length);
        pages_of[threadIdx.x] = (length + p.page_size - 1) / p.page_size;
    }
    __syncthreads();
    int most = 0, limit = 0; /* pages of any row; of any row of this thread's row's sequence */
    for (int i = 0; i < rows; i++) {
        most = max(most, pages_of[i]);
        if (int(threadIdx.x) < rows && sequence_of[i] == sequence_of[threadIdx.x])
            limit = max(limit, pages_of[i]);
    }
    if (int(threadIdx.x) < rows) {
        /* rows of one product and one sequence, from this one on */
        int end = int(threadIdx.x) + 1, top = pages_of[threadIdx.x];
        for (; end < rows && (end & (together - 1)) != 0 && sequence_of[end] == sequence_of[threadIdx.x]; end++)
            top = max(top, pages_of[end]);
        limit_of[threadIdx.x] = limit;
        run_end[threadIdx.x] = end;
        run_pages[threadIdx.x] = top;
    }
    __syncthreads();
    if (!kFused && j_from >= most)
        return;

    uint4 bound[2][KC];
    float scale[2];
    bool there[2];
    int held = -1, held_j = -1; /* whose bounds these are */
    auto hold = [&](int i, int j0) {
        const int s = sequence_of[i], to = limit_of[i];
        held = s;
        held_j = j0;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int j = j0 + g + 8 * h;
            const int page = j < to ? lookup(p, s, j) : -1;
            there[h] = page >= 0;
            const int64_t at = int64_t(page) * p.kv_heads + head;
            const uint4 *b = reinterpret_cast<const uint4 *>(p.bounds + at * 2 * D);
            scale[h] = there[h] ? p.bound_scales[at] : 0.0f;
#pragma unroll
            for (int c = 0; c < KC; c++)
                bound[h][c] = there[h] && c * 4 + t < D / 8 ? b[c * 4 + t] : make_uint4(0, 0, 0, 0);
        }
    };
    hold(0, j_from + warp * kPages);

    for (int gq = 0; gq < p.group; gq += kHeads) {
        const int heads = min(kHeads, p.group - gq);
        if (gq > 0)
            __syncthreads();
        /* queries in 8 bits, a warp for each (row, head): [max(x, 0) |
         * min(x, 0)], and their units; what lies behind meets zeros */
        const int pairs = rows << shift;
        for (int b = warp; b < pairs; b += kWarps * kBatch) {
            float v[kBatch][KC]; /* KC * 64 bytes are KC * 32 dims */
#pragma unroll
            for (int i = 0; i < kBatch; i++) {
                const int pair = b + i * kWarps, row = pair >> shift, h = pair & (span - 1);
                const R *q = static_cast<const R *>(a.q) + int64_t(row0 + row) * a.q_stride +
                             int64_t(head * p.group + gq + h) * D;
#pragma unroll
                for (int c = 0; c < KC; c++) {
                    const int d = lane + 32 * c;
                    v[i][c] = pair < pairs && h < heads && d < D ? finite_key(to_float(q[d])) : 0.0f;
                }
            }
#pragma unroll
            for (int i = 0; i < kBatch; i++) {
                const int pair = b + i * kWarps, row = pair >> shift, h = pair & (span - 1);
                if (pair >= pairs || h >= heads)
                    continue;
                float top = 0.0f;
#pragma unroll
                for (int c = 0; c < KC; c++)
                    top = fmaxf(top, fabsf(v[i][c]));
                const float u = unit_of(warp_max(top)), inv = u > 0.0f ? 1.0f / u : 0.0f; /* exact */
                int8_t *out = queries + (row * span + h) * kPitch;
#pragma unroll
                for (int c = 0; c < KC; c++) {
                    const int d = lane + 32 * c;
                    if (d < D) {
                        const int x = int(rintf(v[i][c] * inv));
                        out[d] = int8_t(max(x, 0));
                        out[D + d] = int8_t(min(x, 0));
                    }
                }
                if (lane == 0)
                    units[row * span + h] = u;
            }
        }
        __syncthreads();
        for (int j0 = j_from + warp * kPages; j0 < min(j_to, most); j0 += kWarps * kPages) {
            for (int i = 0, end; i < rows; i = end) {
                end = run_end[i];
                if (j0 >= run_pages[i])
                    continue;
                if (sequence_of[i] != held || j0 != held_j)
                    hold(i, j0);
                const int first = i & -together; /* row of the product's first column */
                int acc[4] = {0, 0, 0, 0};
                const int8_t *x = queries + (first * span + g) * kPitch + t * 16;
#pragma unroll
                for (int c = 0; c < KC; c++) {
                    const uint4 b = *reinterpret_cast<const uint4 *>(x + c * 64);
                    const uint32_t lo[4] = {bound[0][c].x, bound[1][c].x, bound[0][c].y, bound[1][c].y};
                    const uint32_t hi[4] = {bound[0][c].z, bound[1][c].z, bound[0][c].w, bound[1][c].w};
                    mma_s8(acc, lo, b.x, b.y);
                    mma_s8(acc, hi, b.z, b.w);
                }
                /* this lane: pages g and g + 8, columns 2 t and 2 t + 1 */
                const int row = first + (2 * t >> shift), h0 = 2 * t & (span - 1);
                const bool writes = h0 == 0 && row >= i && row < end;
                const int pages = writes ? pages_of[row] : 0;
                const float *unit = units + first * span + 2 * t;
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    float best = h0 < heads ? float(acc[2 * h]) * unit[0] : -INFINITY;
                    if (h0 + 1 < heads)
                        best = fmaxf(best, float(acc[2 * h + 1]) * unit[1]);
                    if (span > 2)
                        best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, 1));
                    if (span > 4)
                        best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, 2));
                    const int j = j0 + g + 8 * h;
                    if (j < pages) {
                        float *to = kFused ? kept + row * kFusedPages + j
                                           : a.scores + (int64_t(row0 + row) * p.kv_heads + head) * p.max_pages + j;
                        /* beyond fp32's range (pages with infinite keys): below the pages that are always read */
                        float v = there[h] ? fminf(fmaxf(best * scale[h], -kMostFloat), kMostFloat) : -INFINITY;
                        if (gq > 0)
                            v = fmaxf(v, *to);
                        if (j < a.sink_pages || j >= pages - a.recent_pages)
                            v = INFINITY;
                        else if (!there[h])
                            paged_fail(p, kPagedBadPage);
                        *to = v;
                    }
                }
            }
        }
    }
    if constexpr (kFused) {
        static_assert(kWarps >= kMostRows, "a warp for each row");
        __syncthreads();
        if (warp < rows) {
            int32_t *out = a.selected + (int64_t(row0 + warp) * p.kv_heads + head) * a.n_selected;
            const float *score = kept + warp * kFusedPages;
            if (pages_of[warp] <= kFusedPages / 4)
                choose_in_warp<kFusedPages / 128>(score, pages_of[warp], a.n_selected, out);
            else
                choose_in_warp<kFusedPages / 32>(score, pages_of[warp], a.n_selected, out);
        }
    }
}

struct PageKeys {
    const float *score;
    template <int N> __device__ __forceinline__ void own(int i, int there, uint32_t (&k)[N]) const {
        float v[N];
        load_own(score + i, there, v);
#pragma unroll
        for (int e = 0; e < N; e++)
            k[e] = e < there ? ordered_bits(v[e]) : 0u;
    }
};

__global__ void __launch_bounds__(kChooseThreads)
    choose_pages_kernel(const __grid_constant__ PagedSelect a) {
    __shared__ ChooseScratch scratch;
    const PagedPool &p = a.p;
    const int head = blockIdx.x, r = blockIdx.y, tid = threadIdx.x;
    int length;
    begin_kernel();
    row_span(p, a.row_sequence, a.row_length, r, length);
    const int pages = (length + p.page_size - 1) / p.page_size;
    const int64_t at = int64_t(r) * p.kv_heads + head;
    const PageKeys key{a.scores + at * p.max_pages};
    int32_t *out = a.selected + at * a.n_selected;
    uint32_t first[kOwn], threshold;
    int quota;
    own_keys(key, 0, pages, first);
    choose_largest<1>(key, pages, pages, a.n_selected, first, scratch, threshold, quota);
    int ties = 0, n = 0;
    for (int base = 0; base < pages; base += kChooseChunk) {
        uint32_t k[kOwn];
        if (base == 0) {
#pragma unroll
            for (int e = 0; e < kOwn; e++)
                k[e] = first[e];
        } else {
            own_keys(key, base, pages, k);
        }
        const int i0 = base + tid * kOwn;
        int mine = 0, total;
#pragma unroll
        for (int e = 0; e < kOwn; e++)
            mine += i0 + e < pages && k[e] == threshold;
        int rank = ties + block_before(mine, scratch, 0, total);
        ties += total;
        uint32_t chosen = 0;
#pragma unroll
        for (int e = 0; e < kOwn; e++)
            if (i0 + e < pages && (k[e] > threshold || (k[e] == threshold && rank++ < quota)))
                chosen |= 1u << e;
        int to = n + block_before(__popc(chosen), scratch, 1, total);
        n += total;
        for (; chosen; chosen &= chosen - 1)
            out[to++] = i0 + __ffs(chosen) - 1;
    }
    for (int i = n + tid; i < a.n_selected; i += kChooseThreads)
        out[i] = -1;
}

/* The same for at most 128 N pages, N neighbouring ones a thread: for 1024
 * pages, 256 times over, the other form takes 7.8 us and this one 5.8. */
constexpr int kFewThreads = kFewWarps * 32;

template <int N>
__global__ void __launch_bounds__(kFewThreads)
    choose_few_pages_kernel(const __grid_constant__ PagedSelect a) {
    __shared__ int2 counts[2][kFewWarps];
    __shared__ int scans[2][kFewWarps];
    const PagedPool &p = a.p;
    const int head = blockIdx.x, r = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int length;
    begin_kernel();
    row_span(p, a.row_sequence, a.row_length, r, length);
    const int pages = (length + p.page_size - 1) / p.page_size, want = min(a.n_selected, pages);
    const int64_t at = int64_t(r) * p.kv_heads + head;
    int32_t *out = a.selected + at * a.n_selected;
    const PageKeys key{a.scores + at * p.max_pages};
    uint32_t k[N], threshold = 0;
    const int i0 = tid * N, there = max(0, min(N, pages - i0));
    key.own(i0, there, k);
    int quota = want;
    if (want < pages) {
        FewSums sum{counts};
        search_largest(k, want, sum, threshold, quota);
    }
    auto before = [&](int count, int turn) {
        int upto = count;
#pragma unroll
        for (int x = 1; x < 32; x <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, upto, x);
            upto += lane >= x ? v : 0;
        }
        if (lane == 31)
            scans[turn][warp] = upto;
        __syncthreads();
        int less = upto - count;
#pragma unroll
        for (int w = 0; w < kFewWarps; w++)
            less += w < warp ? scans[turn][w] : 0;
        return less;
    };
    int ties = 0;
#pragma unroll
    for (int e = 0; e < N; e++)
        ties += e < there && k[e] == threshold;
    int rank = before(ties, 0);
    uint32_t chosen = 0;
#pragma unroll
    for (int e = 0; e < N; e++)
        if (e < there && (k[e] > threshold || (k[e] == threshold && rank++ < quota)))
            chosen |= 1u << e;
    for (int to = before(__popc(chosen), 1); chosen; chosen &= chosen - 1)
        out[to++] = i0 + __ffs(chosen) - 1;
    for (int i = want + tid; i < a.n_selected; i += kFewThreads)
        out[i] = -1;
}

template <typename R, int KC> cudaError_t launch_scores(const PagedSelect &a, cudaStream_t s) {
    const PagedPool &p = a.p;
    /* rows that may share a sequence share its bounds in registers */
    const int rows_each = a.row_sequence ? kMostRows : 1;
    const int bytes = max(rows_each << columns_of(p.group), kHeads) * (KC * 64 + 64);
    if (p.max_pages <= kFusedPages) {
        const auto kernel = score_kernel<R, KC, true>;
        /* 8 rows of more than 4 heads of more than 128 dims take 52 KB */
        constexpr int kMostBytes = kMostRows * (kHeads * (KC * 64 + 64) + kFusedPages * 4);
        if constexpr (kMostBytes > 40 * 1024) {
            static bool raised[kMaxDevices] = {};
            int device = 0;
            cudaError_t e = cudaGetDevice(&device);
            if (e == cudaSuccess && !raised[device % kMaxDevices])
                e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostBytes);
            if (e != cudaSuccess)
                return e;
            raised[device % kMaxDevices] = true;
        }
        return launch_kernel(kernel, dim3(1, p.kv_heads, (a.rows + rows_each - 1) / rows_each), kWarps * 32,
                             bytes + rows_each * kFusedPages * 4, s, 1, a, rows_each, kFusedPages);
    }
    /* a block's queries are made once for all of its pages: as many of them
     * as still leave two blocks for each SM (36 against 51 us with 128) */
    int pages_each = kWarps * kPages * 4;
    const int row_blocks = (a.rows + rows_each - 1) / rows_each;
    const auto chunks = [&] { return (p.max_pages + pages_each - 1) / pages_each; };
    while (pages_each > kWarps * kPages && int64_t(chunks()) * p.kv_heads * row_blocks < 2 * kMaxSms)
        pages_each /= 2;
    return launch_kernel(score_kernel<R, KC, false>, dim3(chunks(), p.kv_heads, row_blocks), kWarps * 32, bytes, s, 1, a,
                         rows_each, pages_each);
}

template <typename R> cudaError_t scores(const PagedSelect &a, cudaStream_t s) {
    const int D = a.p.head_dim;
    return D <= 32    ? launch_scores<R, 1>(a, s)
           : D <= 64  ? launch_scores<R, 2>(a, s)
           : D <= 96  ? launch_scores<R, 3>(a, s)
           : D <= 128 ? launch_scores<R, 4>(a, s)
                      : launch_scores<R, 8>(a, s);
}

} // namespace

cudaError_t paged_select(const PagedSelect &a, cudaStream_t s) {
    const PagedPool &p = a.p;
    const cudaError_t e = a.type == 0   ? scores<float>(a, s)
                          : a.type == 1 ? scores<__half>(a, s)
                                        : scores<__nv_bfloat16>(a, s);
    if (e != cudaSuccess)
        return e;
    if (p.max_pages <= kFusedPages)
        return cudaSuccess;
    const dim3 items(p.kv_heads, a.rows);
    if (p.max_pages <= 8 * kFewThreads)
        return launch_kernel(choose_few_pages_kernel<8>, items, kFewThreads, 0, s, 1, a);
    return launch_kernel(choose_pages_kernel, items, kChooseThreads, 0, s, 1, a);
}

} // namespace nut
