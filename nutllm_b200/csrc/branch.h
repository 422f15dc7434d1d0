#pragma once
/* Pages of branching sequences (nut_pages_*) and beam selection (nut_beam_*):
 * what the kernels see, and their host-side launchers. */
#include <cstdint>
#include <cuda_runtime.h>

namespace nut {

/* Bits of a page book's error word. */
enum PagesError {
    kPagesBadArgument = 1, /* parent, keep or add */
    kPagesBadLength = 2,   /* a length, or one that the table cannot hold */
    kPagesBadPage = 4,     /* a page number, or a book that contradicts itself */
    kPagesNoneFree = 8
};

constexpr int kPagesMostWarps = 16 * 32; /* of an update */

struct PagesUpdate {
    int32_t *table, *lengths, *refs, *free_pages, *free_count;
    const int32_t *parent, *keep, *add;
    int32_t *copy_from, *copy_to, *copy_slots;
    int sequences, max_pages, n_pages, page_size;
    int32_t *staged;                  /* [sequences][max_pages]: the table to be, */
    int32_t *changes;                 /* from this entry of a sequence on; those before stay */
    int4 *plan;                       /* [sequences]: kept slots, new length, written tail page or -1, parent */
    int32_t *delta, *writers, *first; /* [n_pages], 0 between calls */
    int32_t *freed;                   /* [kPagesMostWarps]: pages given back in each warp's run */
    int32_t *met;                     /* what this call met */
    int32_t *error;                   /* what the handle's calls met */
};
cudaError_t pages_update(const PagesUpdate &a, cudaStream_t s);

constexpr int kBeamTile = 1024; /* logits that a warp takes at a time */
constexpr int kBeamMostOut = 64;

/* A run's sum of exp(logit - top) and its greatest logit. */
struct BeamPart {
    double sum;
    float top;
};

struct BeamSelect {
    const void *logits;
    int64_t stride;
    const float *scores;
    const uint8_t *finished;
    float *out_scores;
    int32_t *out_rows, *out_tokens;
    uint8_t *out_finished;
    int sequences, beams, vocab, n_out, eos, type;
    int runs, run_tiles; /* runs of a row, tiles of a run */
    BeamPart *parts;     /* [rows][runs] */
    unsigned long long *best; /* [rows][runs][n_out], argmax keys, descending, 0 behind them */
};
cudaError_t beam_select(const BeamSelect &a, cudaStream_t s);

} // namespace nut
