#pragma once
/* How the tree attention's kernels share their work (paged_tree.cu,
 * paged_tree_tc.cu).
 *
 * An item is a sequence, a kv head and a block of up to kBlockRows rows; a row
 * is (drafted token, query head of the group), rows of one token together.
 * An item's slots are cut into tiles; all tiles of all items form one line
 * that is cut evenly among the CTAs, whatever the lengths.  An item that lies
 * in one CTA is finished there; of one that spans several each leaves its
 * unnormalised outputs, maxima and sums, which join_kernel puts together in
 * order of the slots: results do not depend on timing. */
#include <cstdint>
#include <cuda_runtime.h>

#include "paged.cuh"

namespace nut {

constexpr float kTreeLog2e = 1.4426950408889634f, kTreeLn2 = 0.6931471805599453f;
constexpr int kTreeTile = 64; /* slots of a tile */
/* What an item costs besides its tiles, in tiles: its queries' way in and its
 * outputs' way out.  With 2, 4 and 6, us in a graph:
 *   32 bf16 caches of 1,024 to 4,096 slots, 16 tokens, 32/8 heads of 128   81.0   78.3   79.7
 *   16 fp16 of 500 to 2,000, 64 tokens, 32/4 of 128                        68.4   63.8   62.7
 *   256 fp16 of 125 to 500, 4 tokens, 32/8 of 64                            152    145    145
 *   4 fp32 of 250 to 1,000, 12 tokens, 32/32 of 128                         45.2   51.2   50.4
 *   24 bf16 of 500 to 2,000, 16 tokens, 4/4 of 256 (fp32 arithmetic)        324    342    363 */
constexpr int kTreeItemCost = 4;
/* The least share of a CTA: each part of an item is written and read again.
 * With 1, 2, 3, 4 and 8, us in a graph:
 *   one bf16 cache of 300 slots, 8 tokens, 32/8 heads of 128   15.1   15.1   15.6   16.6   20.2
 *   2,000 slots, 25 tokens                                     24.8   20.4   20.5   21.3   26.2
 *   4 fp16 of 250 to 1,000, 8 fp32 rows, 32/4 of 64            18.7   18.7   19.3   20.2   24.8
 *   one fp32 of 1,000, 8 tokens, 32/4 of 64                    19.6   19.5   22.5   26.1   40.4
 * (16,000 slots and more, or 32 sequences: no difference) */
constexpr int kTreeLeastShare = 2;

/* The drafted tokens of a sequence and what they see. */
struct TreeSpan {
    int row0, n, prefix, length; /* n = 0: nothing to do */
    bool blind;                  /* its rows see nothing */
};

__device__ __forceinline__ TreeSpan tree_span(const PagedTree &a, int s) {
    const int r0 = a.starts[s], r1 = a.starts[s + 1], stored = a.p.lengths[s];
    TreeSpan x{r0, 0, 0, 0, false};
    if (r0 < 0 || r1 < r0 || r1 > a.rows) {
        paged_fail(a.p, kPagedBadStarts);
        return x;
    }
    x.n = r1 - r0;
    if (x.n == 0)
        return x;
    x.length = checked_length(a.p, stored);
    x.prefix = x.length - x.n;
    if (x.n > a.max_new || x.prefix < 0) {
        if (x.length == stored)
            paged_fail(a.p, kPagedBadStarts);
        x.blind = true;
    }
    return x;
}

__device__ __forceinline__ int tree_tiles(const TreeSpan &x, int tile) { return (x.length + tile - 1) / tile; }

struct TreeItem {
    TreeSpan span;
    int sequence, head;
    int first_row, rows; /* of the sequence's n * group */
    int tiles, tile0, tile1;
    int first; /* where its first tile lies on the line */
    __device__ __forceinline__ bool whole() const { return tile0 == 0 && tile1 == tiles; }
};

/* Walks the items of a share. */
struct TreeCursor {
    int pos, last, s, in_s; /* place on the line, its end, sequence, place within the sequence's */

    __device__ __forceinline__ bool next(const PagedTree &a, int tile, int block_rows, TreeItem &x) {
        while (pos < last) {
            x.span = tree_span(a, s);
            x.sequence = s;
            if (x.span.n == 0 || x.span.blind) {
                s++;
                continue;
            }
            const int all = x.span.n * a.p.group, blocks = (all + block_rows - 1) / block_rows;
            x.tiles = tree_tiles(x.span, tile);
            const int len = x.tiles + kTreeItemCost;
            const int index = in_s / len, place = in_s - index * len;
            const int taken = min(len - place, last - pos);
            x.head = index / blocks;
            x.first_row = (index - x.head * blocks) * block_rows;
            x.rows = min(block_rows, all - x.first_row);
            x.tile0 = max(place - kTreeItemCost, 0);
            x.tile1 = place + taken - kTreeItemCost;
            x.first = pos - place + kTreeItemCost;
            pos += taken;
            in_s += taken;
            if (in_s >= len * a.p.kv_heads * blocks) {
                in_s = 0;
                s++;
            }
            if (x.tile1 > x.tile0)
                return true;
        }
        return false;
    }
};

/* Places of sequence s on the line. */
__device__ __forceinline__ int tree_places(const PagedTree &a, int s, int tile, int block_rows) {
    const TreeSpan x = tree_span(a, s);
    if (x.n == 0 || x.blind)
        return 0;
    return (tree_tiles(x, tile) + kTreeItemCost) * a.p.kv_heads * ((x.n * a.p.group + block_rows - 1) / block_rows);
}

/* This CTA's share of the line; run by all of its kThreads threads. */
template <int kThreads>
__device__ __forceinline__ TreeCursor tree_share(const PagedTree &a, int tile, int block_rows, int &share) {
    __shared__ int sums[kThreads / 32], found[2];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int run = (a.p.sequences + kThreads - 1) / kThreads;
    const int s0 = min(tid * run, a.p.sequences), s1 = min(s0 + run, a.p.sequences);
    int mine = 0;
#pragma unroll 1
    for (int s = s0; s < s1; s++)
        mine += tree_places(a, s, tile, block_rows);
    int upto = mine;
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, upto, x);
        upto += lane >= x ? v : 0;
    }
    if (lane == 31)
        sums[warp] = upto;
    if (tid == 0)
        found[0] = found[1] = 0;
    __syncthreads();
    int total = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 32; w++) {
        upto += w < warp ? sums[w] : 0;
        total += sums[w];
    }
    share = max((total + int(gridDim.x) - 1) / int(gridDim.x), kTreeLeastShare);
    const int start = min(int64_t(blockIdx.x) * share, int64_t(total));
    int at = upto - mine;
    if (start < total && start >= at && start < upto)
#pragma unroll 1
        for (int s = s0; s < s1; s++) {
            const int n = run == 1 ? mine : tree_places(a, s, tile, block_rows);
            if (start < at + n) {
                found[0] = s;
                found[1] = start - at;
                break;
            }
            at += n;
        }
    __syncthreads();
    return {start, min(start + share, total), found[0], found[1]};
}

/* Rows that see nothing; run by `threads` threads of every CTA. */
template <typename R> __device__ __noinline__ void tree_blind_rows(const PagedTree &a, int tid, int threads) {
    const int H = a.p.heads, width = H * a.p.head_dim;
    for (int s = blockIdx.x; s < a.p.sequences; s += gridDim.x) {
        const TreeSpan x = tree_span(a, s);
        if (x.n == 0 || !x.blind)
            continue;
        for (int r = x.row0; r < x.row0 + x.n; r++) {
            for (int i = tid; i < width; i += threads)
                static_cast<R *>(a.out)[r * a.out_stride + i] = from_float<R>(0.0f);
            if (a.lse)
                for (int h = tid; h < H; h += threads)
                    a.lse[int64_t(r) * H + h] = -INFINITY;
        }
    }
}

/* Drafted token of row f of a sequence and kv head. */
__device__ __forceinline__ int tree_node(const PagedTree &a, int f) {
    return int((uint64_t(unsigned(f)) * a.group_magic) >> a.group_shift);
}

/* Row f of a sequence and kv head: its row in q and out, and its query head. */
__device__ __forceinline__ void tree_row(const PagedTree &a, int row0, int head, int f, int64_t &row, int &query_head) {
    const int node = tree_node(a, f);
    row = row0 + node;
    query_head = head * a.p.group + f - node * a.p.group;
}

/* A CTA's part of an item: maxima and sums of its rows, then outputs.  Sums and
 * outputs are those of weights 2^(logit - maximum - rest), times a power of two
 * that all parts share: a rest holds what rounding took from a great maximum.  The item that a CTA's share begins
 * within lies in its first place, another in the second. */
struct TreePart {
    float *maxima, *rests, *sums, *out;
};
__device__ __forceinline__ TreePart tree_part(const PagedTree &a, int cta, int second, int rows) {
    float *at = a.partial + (int64_t(cta) * 2 + second) * a.part_floats;
    return {at, at + rows, at + rows * 2, at + (rows * 3 + 3) / 4 * 4};
}

/* What join_kernel has to know of the item that begins in this CTA and goes on
 * in others; nothing for a CTA without one. */
__device__ __forceinline__ int4 tree_join(const TreeItem &x, int share) {
    const int c0 = x.first / share, c1 = (x.first + x.tiles - 1) / share;
    const int inside = x.first > c0 * share;
    return make_int4(c1 - c0 + 1, x.sequence, x.head, x.first_row * 2 + inside);
}

/* Bit j of the result: whether the row with these mask words sees drafted
 * token base + j (every slot below 0 is the prefix), of n there are. */
__device__ __forceinline__ uint32_t tree_sees(const uint32_t *words, int base, int n) {
    uint32_t bits = 0;
    if (base > -32 && base < n) {
        const int w = base >> 5, shift = base & 31; /* floors */
        const int last = (n - 1) >> 5;
        const uint32_t tail = n & 31 ? (1u << (n & 31)) - 1u : ~0u;
        uint32_t lo = w >= 0 ? words[w] : 0u, hi = w + 1 <= last ? words[w + 1] : 0u;
        if (w == last)
            lo &= tail;
        if (w + 1 == last)
            hi &= tail;
        bits = __funnelshift_r(lo, hi, shift);
    }
    if (base < 0)
        bits |= base <= -32 ? ~0u : (1u << -base) - 1u;
    return bits;
}

/* drop: the inverse of the power of two in the parts' sums. */
cudaError_t tree_join_parts(const PagedTree &a, int ctas, int block_rows, float drop, cudaStream_t s);

} // namespace nut
