/* Attention of drafted tokens over the paged KV cache
 * (nut_paged_tree_attention): fp32 arithmetic on any types, and the joining of
 * split items.
 *
 *   z_t = scale q . k_t,  m = max z,  l = sum exp(z_t - m),
 *   out = sum exp(z_t - m) v_t / l,   lse = m + log l
 * over the slots a row sees, in one pass with a running maximum and sum.
 *
 * A tile is 64 slots, read once for all of an item's rows, in fp32 in shared
 * memory; 256 threads form the products, then the softmax, then the outputs.
 * The next tile's keys are on their way from when the logits are formed, its
 * values from when the outputs are, its pages' numbers a tile before that.
 * What bounds it is that these steps follow one another behind barriers, with
 * two blocks an SM to fill the gaps: of some 11,500 cycles a tile the logits
 * take 3,500, the outputs 2,600 and the softmax 2,700, where FFMA alone would
 * need 2,050.  4 fp32 caches up to 1,000 slots, 32 kv heads of 128 dims, 12
 * tokens (84 MB) 56 us, 1.5 TB/s.  Without the prefetch it was 108 us; a bulk
 * copy a row in place of 16 bytes a thread made no difference at 128 dims and
 * took 29 us in place of 23 at 64.  16-bit caches take it only where the tensor
 * cores' kernel has no form, head_dim above 128: the batch of that kernel's
 * comment was 865 us in a first form of this one.
 */
#include <algorithm>
#include <cstdint>
#include <type_traits>
#include <cuda_runtime.h>

#include "paged_tree.cuh"

namespace nut {
namespace {

constexpr int kThreads = 256;
constexpr int kTile = kTreeTile;

/* kRows: 16, 32 or 64 rows of an item.  Of the logits a thread forms 4 rows by
 * 4 slots over a part of the dims, of the outputs 4 rows by 2 (or more) 4-dim
 * pieces over a part of the slots: fewer operands out of shared memory than
 * smaller tiles over all of them.  Neighbouring lanes have the other parts. */
template <int kRows, int DP> struct WidePlan {
    static constexpr int kAcross = kThreads / (kRows / 4); /* threads that share 4 rows */
    static constexpr int kSplits = kAcross / (kTile / 4);  /* of the dims */
    static constexpr int kPieces = kRows * DP / 16 / kThreads > 2 ? kRows * DP / 16 / kThreads : 2;
    static constexpr int kEvery = DP / 4 / kPieces;        /* pieces between a thread's */
    static constexpr int kShares = kAcross / kEvery;       /* of the slots */
    /* floats between rows, so that 8 neighbouring lanes meet no bank twice: they are kSplits pieces
     * of 8 / kSplits keys, and 8 / kShares pieces of kShares values */
    static constexpr int kKeyPitch = DP + 4 * kSplits, kValuePitch = DP + (kShares > 1 ? 32 / kShares : 4);
    static constexpr int kWeights = kRows + 4; /* of a slot */
    static constexpr int kFloats = (kRows + kTile) * kKeyPitch + kTile * (kValuePitch + kWeights);
    static constexpr int kBytes = kFloats * 4;
    static constexpr int kOfRow = kThreads / kRows; /* threads of a row's softmax */
    static constexpr int kPerSm = kBytes <= 110 * 1024 ? 2 : 1;
    static_assert(kSplits >= 1 && kSplits <= 4 && kShares >= 1 && kShares <= 8, "lanes of a part lie in a warp");
    static_assert(kShares <= 4 || kShares == 4 * kPieces, "each lane writes a row, or a piece of it");
};

/* Two products added to two sums in one instruction. */
__device__ __forceinline__ void add_products(Two &sum, Two a, Two b) {
    asm("fma.rn.f32x2 %0, %1, %2, %0;\n" : "+l"(sum) : "l"(a), "l"(b));
}

/* 16 bytes to shared memory, or zeros. */
__device__ __forceinline__ void copy_piece(float *to, const void *from, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(uint32_t(__cvta_generic_to_shared(to))), "l"(from),
                 "r"(there ? 16 : 0)
                 : "memory");
}
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
/* All but the newest group of copies. */
__device__ __forceinline__ void await_copies() { asm volatile("cp.async.wait_group 1;\n" ::: "memory"); }

template <typename T> __device__ __forceinline__ void load_four(const T *x, float *v) {
    if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4 *>(v) = *reinterpret_cast<const float4 *>(x);
    } else {
        const uint2 a = *reinterpret_cast<const uint2 *>(x);
        const T *e = reinterpret_cast<const T *>(&a);
#pragma unroll
        for (int i = 0; i < 4; i++)
            v[i] = to_float(e[i]);
    }
}

template <int kRows, int DP, typename T, typename R>
__global__ void __launch_bounds__(kThreads, (WidePlan<kRows, DP>::kPerSm)) wide_kernel(const __grid_constant__ PagedTree a) {
    using W = WidePlan<kRows, DP>;
    extern __shared__ float4 smem_raw[];
    float *queries = reinterpret_cast<float *>(smem_raw), *keys = queries + kRows * W::kKeyPitch,
          *values = keys + kTile * W::kKeyPitch, *weights = values + kTile * W::kValuePitch; /* [slot][row] */
    __shared__ int64_t places[2][kTile]; /* elements from the pool's start, -1: no such slot */
    __shared__ float maxima[kRows], sums[kRows], factors[kRows];
    const PagedPool &p = a.p;
    const int tid = threadIdx.x, D = p.head_dim;
    begin_kernel();
    int share;
    TreeCursor cursor = tree_share<kThreads>(a, kTile, kRows, share);
    tree_blind_rows<R>(a, tid, kThreads);
    const int start = cursor.pos;
    const int r0 = tid / W::kAcross * 4, c0 = tid % W::kAcross; /* of the products */
    const int split = c0 % W::kSplits, slot0 = c0 / W::kSplits;
    const int share0 = c0 % W::kShares, piece0 = c0 / W::kShares;
    constexpr int kOfWarp = 32 / W::kOfRow; /* rows of a warp's softmax; rows of neighbouring lanes differ */
    const int soft_row = tid / 32 * kOfWarp + tid % kOfWarp, soft_at = tid % 32 / kOfWarp;
    const float unit = a.scale * kTreeLog2e;
    int4 join = make_int4(0, 0, 0, 0);

    TreeItem x;
    while (cursor.next(a, kTile, kRows, x)) {
        __syncthreads();
        for (int i = tid; i < kRows * (DP / 4); i += kThreads) {
            const int r = i / (DP / 4), d = i % (DP / 4) * 4;
            float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            if (r < x.rows && d < D) {
                int64_t row;
                int h;
                tree_row(a, x.span.row0, x.head, x.first_row + r, row, h);
                const R *q = static_cast<const R *>(a.q) + row * a.q_stride + int64_t(h) * D + d;
#pragma unroll
                for (int j = 0; j < 4; j++)
                    v[j] = to_float(q[j]);
            }
            *reinterpret_cast<float4 *>(queries + r * W::kKeyPitch + d) = make_float4(v[0], v[1], v[2], v[3]);
        }
        if (tid < kRows) {
            maxima[tid] = -INFINITY;
            sums[tid] = 0.0f;
        }
        Two o2[4][W::kPieces][2];
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
            for (int k = 0; k < W::kPieces; k++)
                o2[r][k][0] = o2[r][k][1] = 0;

        /* Threads 0 to 63 have a slot of a tile each: its page is looked up a tile before its place
         * is needed. */
        const auto look = [&](int tile) {
            const int t = tile * kTile + tid;
            return tid < kTile && tile < x.tile1 && t < x.span.length
                       ? p.table[int64_t(x.sequence) * p.max_pages + int((uint64_t(unsigned(t)) * a.page_magic) >> a.page_shift)]
                       : -1;
        };
        const auto place = [&](int tile, int page) {
            if (tid < kTile && tile < x.tile1) {
                const int t = tile * kTile + tid;
                int64_t at = -1;
                if (t < x.span.length) {
                    const int j = int((uint64_t(unsigned(t)) * a.page_magic) >> a.page_shift);
                    if (unsigned(page) < unsigned(p.n_pages))
                        at = int64_t(page) * p.page_stride + int64_t(x.head) * p.head_stride +
                             int64_t(t - j * p.page_size) * p.slot_stride;
                    else
                        paged_fail(p, kPagedBadPage);
                }
                places[tile & 1][tid] = at;
            }
        };
        const auto fetch = [&](int tile, const void *pool, float *to, int pitch) {
            if (tile < x.tile1)
                for (int i = tid; i < kTile * (DP / 4); i += kThreads) {
                    const int t = i / (DP / 4), d = i % (DP / 4) * 4;
                    const int64_t at = places[tile & 1][t];
                    const bool there = at >= 0 && d < D;
                    const T *from = static_cast<const T *>(pool) + (there ? at + d : 0);
                    if constexpr (sizeof(T) == 4) {
                        copy_piece(to + t * pitch + d, from, there);
                    } else {
                        float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                        if (there)
                            load_four(from, v);
                        *reinterpret_cast<float4 *>(to + t * pitch + d) = make_float4(v[0], v[1], v[2], v[3]);
                    }
                }
            copies_done();
        };
        place(x.tile0, look(x.tile0));
        int page = look(x.tile0 + 1);
        __syncthreads();
        fetch(x.tile0, p.keys, keys, W::kKeyPitch);
        fetch(x.tile0, p.values, values, W::kValuePitch);
        for (int tile = x.tile0; tile < x.tile1; tile++) {
            const int t0 = tile * kTile;
            place(tile + 1, page);
            page = look(tile + 2);
            await_copies(); /* the keys */
            __syncthreads();
            Two z2[4][4];
#pragma unroll
            for (int r = 0; r < 4; r++)
#pragma unroll
                for (int k = 0; k < 4; k++)
                    z2[r][k] = 0;
#pragma unroll 2
            for (int d = split * 4; d < DP; d += 4 * W::kSplits) {
                ulonglong2 q[4];
#pragma unroll
                for (int r = 0; r < 4; r++)
                    q[r] = *reinterpret_cast<const ulonglong2 *>(queries + (r0 + r) * W::kKeyPitch + d);
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const ulonglong2 c = *reinterpret_cast<const ulonglong2 *>(keys + (slot0 + k * (kTile / 4)) * W::kKeyPitch + d);
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        add_products(z2[r][k], q[r].x, c.x);
                        add_products(z2[r][k], q[r].y, c.y);
                    }
                }
            }
            /* the dims' parts meet: of 4 rows a lane keeps 4 / kSplits */
            constexpr int kKept = 4 / W::kSplits;
            float z[4][4];
#pragma unroll
            for (int r = 0; r < 4; r++)
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const float2 v = parts_of(z2[r][k]);
                    z[r][k] = (v.x + v.y) * unit;
                }
#pragma unroll
            for (int e = W::kSplits / 2, left = 4; e > 0; e >>= 1) {
                left /= 2;
#pragma unroll
                for (int r = 0; r < left; r++)
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const bool upper = split & e;
                        const float kept = upper ? z[r + left][k] : z[r][k], sent = upper ? z[r][k] : z[r + left][k];
                        z[r][k] = kept + __shfl_xor_sync(0xffffffffu, sent, e);
                    }
            }
#pragma unroll
            for (int k = 0; k < 4; k++) {
                float *to = weights + (slot0 + k * (kTile / 4)) * W::kWeights + r0 + split * kKept;
                if constexpr (kKept == 4)
                    *reinterpret_cast<float4 *>(to) = make_float4(z[0][k], z[1][k], z[2][k], z[3][k]);
                else if constexpr (kKept == 2)
                    *reinterpret_cast<float2 *>(to) = make_float2(z[0][k], z[1][k]);
                else
                    *to = z[0][k];
            }
            __syncthreads();
            fetch(tile + 1, p.keys, keys, W::kKeyPitch);

            /* softmax: kOfRow lanes a row, every kOfRow-th slot each */
            constexpr int kEach = kTile / W::kOfRow;
            float *own = weights + soft_at * W::kWeights + soft_row;
            float v[kEach], top = -INFINITY;
            {
                uint32_t sees[2] = {0, 0}; /* of 32 slots from this thread's first on, and of 32 behind them */
                const int base = t0 - x.span.prefix;
                if (soft_row < x.rows) {
                    if (base <= -kTile) {
                        sees[0] = sees[1] = ~0u;
                    } else {
                        const int node = tree_node(a, x.first_row + soft_row);
                        const uint32_t *words = a.mask + (int64_t(x.span.row0) + node) * a.mask_words;
                        sees[0] = tree_sees(words, base + soft_at, x.span.n);
                        sees[1] = tree_sees(words, base + soft_at + 32, x.span.n);
                    }
                }
#pragma unroll
                for (int j = 0; j < kEach; j++) {
                    const int t = j * W::kOfRow;
                    v[j] = ((sees[t / 32] >> (t % 32)) & 1) && places[tile & 1][soft_at + t] >= 0 ? own[t * W::kWeights] : -INFINITY;
                    top = fmaxf(top, v[j]);
                }
            }
#pragma unroll
            for (int e = 16; e >= kOfWarp; e >>= 1)
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, e));
            const float before = maxima[soft_row], next = fmaxf(before, top);
            const float from = next == -INFINITY ? 0.0f : next;
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < kEach; j++) {
                const float w = exp2f(v[j] - from);
                own[j * W::kOfRow * W::kWeights] = v[j] == -INFINITY ? -0.0f : w;
                sum += w;
            }
#pragma unroll
            for (int e = 16; e >= kOfWarp; e >>= 1)
                sum += __shfl_xor_sync(0xffffffffu, sum, e);
            if (soft_at == 0) {
                const float keep = before == next ? 1.0f : exp2f(before - next);
                factors[soft_row] = keep;
                maxima[soft_row] = next;
                sums[soft_row] = sums[soft_row] * keep + sum;
            }
            await_copies(); /* the values */
            __syncthreads();
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const float keep = factors[r0 + r];
#pragma unroll
                for (int k = 0; k < W::kPieces; k++)
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        const float2 v = parts_of(o2[r][k][j]);
                        o2[r][k][j] = two_of(v.x * keep, v.y * keep);
                    }
            }
            /* values that a row does not see may be infinite or NaN: a weight of -0 takes no part.  (One
             * that is seen and weighs 0 beside a much greater one does: 0 times it is NaN.) */
            constexpr Two kUnseen = 0x8000000080000000ull; /* two of -0 */
            const auto multiply = [&](auto drafted) {
#pragma unroll 4
                for (int t = share0; t < kTile; t += W::kShares) {
                    const float4 of = *reinterpret_cast<const float4 *>(weights + t * W::kWeights + r0);
                    const Two w[4] = {two_of(of.x, of.x), two_of(of.y, of.y), two_of(of.z, of.z), two_of(of.w, of.w)};
#pragma unroll
                    for (int k = 0; k < W::kPieces; k++) {
                        const ulonglong2 c =
                            *reinterpret_cast<const ulonglong2 *>(values + t * W::kValuePitch + (piece0 + k * W::kEvery) * 4);
#pragma unroll
                        for (int r = 0; r < 4; r++) {
                            const bool none = decltype(drafted)::value && w[r] == kUnseen;
                            add_products(o2[r][k][0], w[r], none ? 0 : c.x);
                            add_products(o2[r][k][1], w[r], none ? 0 : c.y);
                        }
                    }
                }
            };
            if (t0 + kTile > x.span.prefix)
                multiply(std::true_type());
            else
                multiply(std::false_type());
            __syncthreads();
            fetch(tile + 1, p.values, values, W::kValuePitch);
        }
        float o[4][W::kPieces][4];
#pragma unroll
        for (int r = 0; r < 4; r++)
#pragma unroll
            for (int k = 0; k < W::kPieces; k++)
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const float2 v = parts_of(o2[r][k][j]);
                    o[r][k][2 * j] = v.x;
                    o[r][k][2 * j + 1] = v.y;
                }
#pragma unroll
        for (int e = W::kShares / 2; e > 0; e >>= 1) /* the slots' parts meet */
#pragma unroll
            for (int r = 0; r < 4; r++)
#pragma unroll
                for (int k = 0; k < W::kPieces; k++)
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        o[r][k][j] += __shfl_xor_sync(0xffffffffu, o[r][k][j], e);

        const bool whole = x.whole();
        const TreePart part = tree_part(a, blockIdx.x, x.first <= start ? 0 : 1, x.rows);
        if (tid < x.rows) {
            const float m = maxima[tid], l = sums[tid];
            if (whole) {
                int64_t row;
                int h;
                tree_row(a, x.span.row0, x.head, x.first_row + tid, row, h);
                if (a.lse)
                    a.lse[row * p.heads + h] = l == 0.0f ? -INFINITY : (m + log2f(l)) * kTreeLn2;
            } else {
                part.maxima[tid] = m;
                part.rests[tid] = 0.0f;
                part.sums[tid] = l;
            }
        }
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const int f = r0 + r;
            if (f >= x.rows)
                break;
            if ((r ^ share0) & ((W::kShares < 4 ? W::kShares : 4) - 1)) /* another lane's */
                continue;
            int64_t row;
            int h;
            tree_row(a, x.span.row0, x.head, x.first_row + f, row, h);
            const float inv = !whole ? 1.0f : sums[f] == 0.0f ? 0.0f : 1.0f / sums[f];
#pragma unroll
            for (int k = 0; k < W::kPieces; k++) {
                const int d = (piece0 + k * W::kEvery) * 4;
                if (d >= D)
                    break;
                if (W::kShares > 4 && k != share0 / 4)
                    continue;
                if (whole) {
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        static_cast<R *>(a.out)[row * a.out_stride + int64_t(h) * D + d + j] = output_of<R>(o[r][k][j] * inv);
                } else {
                    *reinterpret_cast<float4 *>(part.out + int64_t(f) * D + d) = make_float4(o[r][k][0], o[r][k][1], o[r][k][2], o[r][k][3]);
                }
            }
        }
        if (!whole && x.tile0 == 0)
            join = tree_join(x, share);
    }
    if (tid == 0)
        a.joins[blockIdx.x] = join;
}

/* ---- joining the parts of an item --------------------------------------- */

constexpr float kNothing = -1.0f; /* the factor of a part in which the row saw nothing */
constexpr int kJoinWarps = 8, kJoinOwn = 2, kJoinRows = kJoinWarps * kJoinOwn;

/* out = sum_c O_c 2^(m_c - m) / sum_c l_c 2^(m_c - m), m_c a maximum and its rest, for two rows a warp, whose loads
 * are in flight together.  Lanes turn the parts' maxima and sums into factors, 32 parts at a time,
 * then take 4 dims each.  It is round trips: which item, its span, maxima, outputs; 8.4 us after 32
 * caches of up to 4,096 slots, 10 with a row a warp, whose blocks came in two waves. */
template <typename R>
__global__ void __launch_bounds__(kJoinWarps * 32, 4) join_kernel(const __grid_constant__ PagedTree a, int block_rows, float drop) {
    begin_kernel();
    const int4 join = a.joins[blockIdx.x];
    const int parts = join.x, lane = threadIdx.x & 31;
    if (parts == 0)
        return;
    const PagedPool &p = a.p;
    const int D = p.head_dim, first_row = join.w >> 1, inside = join.w & 1;
    const int row0 = a.starts[join.y], n = a.starts[join.y + 1] - row0;
    const int rows = min(block_rows, n * p.group - first_row);
    const int f0 = int(blockIdx.y) * kJoinRows + int(threadIdx.x >> 5) * kJoinOwn;
    if (f0 >= rows)
        return;
    const TreePart first = tree_part(a, blockIdx.x, inside, rows), second = tree_part(a, blockIdx.x + 1, 0, rows);
    const int64_t step = 2 * a.part_floats;
    const auto at = [&](const float *x, const float *y, int c, int f) { return (c == 0 ? x : y + (c - 1) * step) + min(f, rows - 1); };
    float from[kJoinOwn], rest[kJoinOwn], sum[kJoinOwn]; /* the greatest maximum, and its greatest rest */
#pragma unroll
    for (int r = 0; r < kJoinOwn; r++) {
        from[r] = rest[r] = -INFINITY;
        sum[r] = 0.0f;
    }
    for (int c = lane; c < parts; c += 32)
#pragma unroll
        for (int r = 0; r < kJoinOwn; r++) {
            const float most = *at(first.maxima, second.maxima, c, f0 + r), more = *at(first.rests, second.rests, c, f0 + r);
            rest[r] = most > from[r] ? more : most == from[r] ? fmaxf(rest[r], more) : rest[r];
            from[r] = fmaxf(from[r], most);
        }
#pragma unroll
    for (int r = 0; r < kJoinOwn; r++) {
        const float most = warp_max(from[r]);
        rest[r] = warp_max(from[r] == most ? rest[r] : -INFINITY);
        from[r] = most;
        if (most == -INFINITY)
            from[r] = rest[r] = 0.0f;
    }
    constexpr int kMost = 2; /* pieces of 4 dims a lane, 128 dims apart */
    float4 o[kJoinOwn][kMost];
#pragma unroll
    for (int r = 0; r < kJoinOwn; r++)
#pragma unroll
        for (int k = 0; k < kMost; k++)
            o[r][k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int c0 = 0; c0 < parts; c0 += 32) {
        const int c = c0 + lane, many = min(32, parts - c0);
        float factor[kJoinOwn];
#pragma unroll
        for (int r = 0; r < kJoinOwn; r++) {
            const float most = c < parts ? *at(first.maxima, second.maxima, c, f0 + r) : -INFINITY;
            const float more = c < parts ? *at(first.rests, second.rests, c, f0 + r) : 0.0f;
            factor[r] = exp2f((most - from[r]) + (more - rest[r]));
            sum[r] += c < parts ? *at(first.sums, second.sums, c, f0 + r) * factor[r] : 0.0f;
            if (most == -INFINITY)
                factor[r] = kNothing;
        }
#pragma unroll
        for (int k = 0; k < kMost; k++) {
            if (k * 128 >= D)
                break;
            const int d = k * 128 + lane * 4;
            constexpr int kFlight = 4;
            for (int i0 = 0; i0 < many; i0 += kFlight) {
                float4 v[kFlight][kJoinOwn];
#pragma unroll
                for (int i = 0; i < kFlight; i++) {
                    const int part = c0 + i0 + i;
                    const float *x = (part == 0 ? first.out : second.out + (part - 1) * step) + d;
#pragma unroll
                    for (int r = 0; r < kJoinOwn; r++)
                        v[i][r] = i0 + i < many && d < D
                                      ? *reinterpret_cast<const float4 *>(x + min(f0 + r, rows - 1) * D)
                                      : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                }
#pragma unroll
                for (int i = 0; i < kFlight; i++)
#pragma unroll
                    for (int r = 0; r < kJoinOwn; r++) {
                        const float w = __shfl_sync(0xffffffffu, factor[r], i0 + i);
                        /* (0, beside a much greater maximum: infinities and NaN of that part become NaN) */
                        if (w != kNothing) {
                            o[r][k].x = fmaf(v[i][r].x, w, o[r][k].x);
                            o[r][k].y = fmaf(v[i][r].y, w, o[r][k].y);
                            o[r][k].z = fmaf(v[i][r].z, w, o[r][k].z);
                            o[r][k].w = fmaf(v[i][r].w, w, o[r][k].w);
                        }
                    }
            }
        }
    }
#pragma unroll
    for (int r = 0; r < kJoinOwn; r++) {
        const float all = warp_sum(sum[r]), inv = all == 0.0f ? 0.0f : 1.0f / all;
        if (f0 + r >= rows)
            break;
        int64_t row;
        int h;
        tree_row(a, row0, join.z, first_row + f0 + r, row, h);
        if (a.lse && lane == 0)
            a.lse[row * p.heads + h] = all == 0.0f ? -INFINITY : (from[r] + (rest[r] + log2f(all * drop))) * kTreeLn2;
        R *to = static_cast<R *>(a.out) + row * a.out_stride + int64_t(h) * D;
#pragma unroll
        for (int k = 0; k < kMost; k++) {
            const int d = k * 128 + lane * 4;
            if (d < D) {
                const R e[4] = {output_of<R>(o[r][k].x * inv), output_of<R>(o[r][k].y * inv), output_of<R>(o[r][k].z * inv),
                                output_of<R>(o[r][k].w * inv)};
                if (a.aligned) {
                    if constexpr (sizeof(R) == 4)
                        *reinterpret_cast<float4 *>(to + d) = make_float4(e[0], e[1], e[2], e[3]);
                    else
                        *reinterpret_cast<uint2 *>(to + d) = *reinterpret_cast<const uint2 *>(e);
                } else {
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        to[d + j] = e[j];
                }
            }
        }
    }
}

template <int kRows, int DP, typename T, typename R> cudaError_t launch_wide(const PagedTree &a, cudaStream_t s) {
    using W = WidePlan<kRows, DP>;
    const auto kernel = wide_kernel<kRows, DP, T, R>;
    static bool set[kMaxDevices] = {};
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess)
        return e;
    if (!set[device % kMaxDevices]) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, W::kBytes);
        if (e != cudaSuccess)
            return e;
        set[device % kMaxDevices] = true;
    }
    static_assert(W::kPerSm <= kTreeCtasPerSm, "the workspace has room for as many");
    const int ctas = a.sms * W::kPerSm;
    e = launch_kernel(kernel, dim3(ctas), kThreads, W::kBytes, s, 1, a);
    return e != cudaSuccess ? e : tree_join_parts(a, ctas, kRows, 1.0f, s);
}

/* Rows of an item, by how many a sequence can have: few that fill them, two blocks an SM; or more of
 * them, between which a tile is shared.  With 16, 32 and 64, us for fp32 caches of 24 sequences up
 * to 2,000 slots, 32 kv heads of 128 dims:
 *   rows    16   48   64   96  128   512
 *   16     336  554  672  934 1203  5726
 *   32     493  578  648  833 1029  4395
 *   64     890  905  921 1095 1251  4384
 * (512 rows of 8 kv heads of 64: 877, 659, 586; of 4 of 256, bf16: 3492, 2161, 1627). */
template <int DP, typename T, typename R> cudaError_t launch_wide(const PagedTree &a, cudaStream_t s) {
    const int64_t rows = int64_t(a.max_new) * a.p.group;
    return rows <= 48    ? launch_wide<16, DP, T, R>(a, s)
           : rows <= 128 ? launch_wide<32, DP, T, R>(a, s)
                         : launch_wide<64, DP, T, R>(a, s);
}

template <typename T, typename R> cudaError_t launch_wide(const PagedTree &a, cudaStream_t s) {
    if constexpr (sizeof(T) == 4) {
        if (a.p.head_dim <= 64)
            return launch_wide<64, T, R>(a, s);
        if (a.p.head_dim <= 128)
            return launch_wide<128, T, R>(a, s);
    }
    return launch_wide<256, T, R>(a, s);
}

} // namespace

cudaError_t tree_join_parts(const PagedTree &a, int ctas, int block_rows, float drop, cudaStream_t s) {
    if (a.p.capacity <= kTreeTile) /* items of one tile lie in one block */
        return cudaSuccess;
    const int rows = int(std::min<int64_t>(block_rows, int64_t(a.max_new) * a.p.group));
    const dim3 grid(ctas, (rows + kJoinRows - 1) / kJoinRows);
    const auto kernel = a.type == 0 ? join_kernel<float> : a.type == 1 ? join_kernel<__half> : join_kernel<__nv_bfloat16>;
    return launch_kernel(kernel, grid, kJoinWarps * 32, 0, s, 1, a, block_rows, drop);
}

int64_t tree_part_floats(const PagedPool &p, int max_new) {
    const int64_t rows = std::min<int64_t>(128, int64_t(max_new) * p.group);
    return (rows * 3 + 3) / 4 * 4 + rows * p.head_dim;
}

int64_t tree_most_places(const PagedPool &p, int max_new, int64_t rows) {
    const int64_t most = std::min<int64_t>(rows, int64_t(p.sequences) * max_new);
    return (most * p.heads / 16 + int64_t(p.sequences) * p.kv_heads + 1) * (p.capacity / 64 + 1 + kTreeItemCost);
}

cudaError_t paged_tree(const PagedTree &a, cudaStream_t s) {
    if (a.p.type != 0 && a.p.head_dim <= 128)
        return paged_tree_tc(a, s);
    if (a.p.type == 0)
        return launch_wide<float, float>(a, s);
    if (a.p.type == 1)
        return a.type == 0 ? launch_wide<__half, float>(a, s) : launch_wide<__half, __half>(a, s);
    return a.type == 0 ? launch_wide<__nv_bfloat16, float>(a, s) : launch_wide<__nv_bfloat16, __nv_bfloat16>(a, s);
}

} // namespace nut
