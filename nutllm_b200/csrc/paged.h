#pragma once
/* Paged KV cache operators (nut_paged_* in nutllm_cuda.h): what the kernels
 * see of a pool, and their host-side launchers. */
#include <cstdint>
#include <cuda.h>
#include <cuda_runtime.h>

namespace nut {

/* Bits of a handle's error word. */
enum PagedError {
    kPagedBadPage = 1,     /* page number outside the pool */
    kPagedBadLength = 2,   /* length outside [0, capacity] */
    kPagedBadSequence = 4, /* row's sequence outside the table */
    kPagedBadStarts = 8,   /* starts not ascending, or more new rows than slots */
    kPagedBadPosition = 16, /* position outside the rotation table */
    kPagedTimeout = 32      /* a copy did not arrive in time */
};

struct PagedPool {
    void *keys, *values;
    const int32_t *table, *lengths;
    int8_t *bounds;
    float *bound_scales;
    int64_t page_stride, head_stride, slot_stride;
    int sequences, max_pages, n_pages, page_size;
    int heads, kv_heads, head_dim, group; /* group = heads / kv_heads */
    int capacity;                         /* max_pages * page_size */
    int type;
    int *error;
};

struct PagedAppend {
    PagedPool p;
    const void *q, *k, *v;
    void *q_out;
    int64_t q_stride, k_stride, v_stride, q_out_stride;
    const int32_t *starts, *seen;
    const float *cos, *sin;
    int rows, max_new, rope_rows, type;
    int32_t *positions;
    float *weights;
    const int32_t *row_position; /* [rows], or NULL: by the slots */
};

struct PagedAttention {
    /* (dim, slot, 128-byte column, kv head, page), in boxes of 16 slots by all
     * columns; where page_size is no multiple of 16 or head_dim none of a
     * column there is but one column, head_dim wide, and boxes are 128 bytes
     * of `box` slots */
    CUtensorMap key_map, value_map;
    PagedPool p;
    int box; /* the greatest power of two up to 16 that divides page_size */
    int whole_columns;
    uint64_t page_magic; /* v / page_size = v * magic >> shift for v < 2^31 */
    int page_shift;
    const void *q;
    void *out;
    int64_t q_stride, out_stride;
    float *lse;
    const int32_t *row_sequence, *row_length, *selected;
    int n_selected;
    const float *weights;
    float *weights_out;
    int rows, type;
    float scale;
    float *logits; /* [sequences][heads][capacity] with weights, in log2 */
    float *lse2;   /* [sequences][heads] with weights, in log2 */
    float *partial; /* [CTAs][2][paged_part_floats]: items shared between CTAs */
    int *counters;  /* [max_rows][items of a row], 0 between calls */
    int sms;
};

/* A CTA's part of an attention item: maxima [8], sums [8], outputs [8][padded dim]. */
constexpr int paged_part_floats(int padded) { return 8 * 2 + 8 * padded; }
constexpr int kMaxCtasPerSm = 3;
constexpr int kMaxSms = 160;
constexpr int kMaxDevices = 64;

struct PagedSelect {
    PagedPool p;
    const void *q;
    int64_t q_stride;
    const int32_t *row_sequence, *row_length;
    int32_t *selected;
    int n_selected, sink_pages, recent_pages, rows, type;
    float *scores; /* [rows][kv_heads][max_pages] */
};

struct PagedEvict {
    PagedPool p;
    const float *weights;
    const int32_t *positions, *seen;
    int budget, sinks, recent;
    int32_t *new_lengths;
    float *weights_out;
    int32_t *positions_out;
    int32_t *pairs;  /* [sequences][kv_heads][capacity]: holes from the start on, sources from the middle on */
    int32_t *counts; /* [sequences][kv_heads][2]: pairs, new length (-1: as it was) */
};

struct PagedCompact {
    PagedPool p;
    const int32_t *starts, *accepted;
    int n_accepted;
    int32_t *new_lengths, *positions;
    float *weights;
    int32_t *order; /* [sequences]: blocks that are through, 0 between calls */
};

struct PagedCopy {
    PagedPool p;
    const int32_t *source, *target, *slots;
    int count;
};

constexpr int kTreeMost = 1024;   /* drafted tokens of a sequence */
constexpr int kTreeMostBox = 64; /* slots of a box of the tree attention's maps */
constexpr int kTreeCtasPerSm = 2;

struct PagedTree {
    /* (dim, slot, 128-byte column, kv head, page) in boxes of one column by
     * `box` slots; the column is the whole row where head_dim is no multiple of
     * it.  wide_value_map: all columns by 16 slots, where there are such */
    CUtensorMap key_map, value_map, wide_value_map;
    PagedPool p;
    int box, whole_columns, aligned; /* aligned: rows of q and out begin at multiples of 16 bytes */
    uint64_t page_magic, group_magic; /* as PagedAttention's */
    int page_shift, group_shift;
    const void *q;
    void *out;
    int64_t q_stride, out_stride;
    float *lse;
    const int32_t *starts;
    const uint32_t *mask;
    int mask_words, rows, max_new, type;
    float scale;
    float *partial; /* [CTAs][2][part_floats] */
    int4 *joins;    /* [CTAs]: the item that begins in a CTA and ends in another */
    int64_t part_floats;
    int sms;
};

/* head_dim as the attention's kernels are made for. */
inline int paged_padded_dim(int type, int D) {
    return type == 0 ? (D <= 32 ? 32 : D <= 64 ? 64 : D <= 128 ? 128 : 256)
                     : (D <= 64 ? 64 : D <= 96 ? 96 : D <= 128 ? 128 : D <= 192 ? 192 : 256);
}
/* What the tree attention's kernels want of a pool (paged_tree.cu): floats of
 * a CTA's part of an item, and the most places on the line of tiles. */
int64_t tree_part_floats(const PagedPool &p, int max_new);
int64_t tree_most_places(const PagedPool &p, int max_new, int64_t rows);

/* 128-byte columns of such a row in shared memory. */
inline int paged_columns(int type, int D) {
    return (paged_padded_dim(type, D) * (type == 0 ? 4 : 2) + 127) / 128;
}

cudaError_t paged_append(const PagedAppend &a, cudaStream_t s);
cudaError_t paged_summarise(const PagedPool &p, cudaStream_t s);
cudaError_t paged_attention(const PagedAttention &a, cudaStream_t s);
cudaError_t paged_select(const PagedSelect &a, cudaStream_t s);
cudaError_t paged_evict(const PagedEvict &a, cudaStream_t s);
cudaError_t paged_compact(const PagedCompact &a, cudaStream_t s);
cudaError_t paged_copy(const PagedCopy &a, cudaStream_t s);
cudaError_t paged_tree(const PagedTree &a, cudaStream_t s);
cudaError_t paged_tree_tc(const PagedTree &a, cudaStream_t s);

} // namespace nut
