/* Beam search's choice over beams and vocabulary (nut_beam_select).
 *
 *   score(b, t) = scores[b] + logit[b][t] - log sum_u exp(logit[b][u])
 * The logits are read once.  A block takes a chunk of 8,192 logits of one
 * beam, 32 in each thread's registers: their maximum, the sum of their
 * exponentials, and the chunk's n_out greatest.  For those each warp finds
 * its ceil(n_out / 8) greatest of its lanes' maxima; the least of what the 8
 * warps found is a threshold that at least n_out logits reach, and few more
 * do.  Those are listed in shared memory and ranked by counting.  (Where equal
 * logits overflow the list, the greatest is taken n_out times.)  Then a block
 * for each request joins its chunks' sums in fp64, turns the candidates into
 * scores and chooses among them the same way.
 *
 * Sums: exponentials and a thread's sum of 32 in fp32, all beyond it in fp64
 * where two chunks meet.  Scores are compared in fp64: a logit is fp32, and
 * in an fp32 sum neighbours of different beams would often round to a tie.
 */
#include <cfloat>
#include <cstdint>
#include <cuda_runtime.h>

#include "branch.h"
#include "paged.cuh"

namespace nut {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kWarps = kBeamThreads / 32;
constexpr int kListed = 1024; /* candidates that are ranked by counting */

/* A logit as it counts: NaN as -infinity, +infinity as the greatest float. */
__device__ __forceinline__ float counted(float v) { return fminf(fmaxf(v, -INFINITY), FLT_MAX); }

/* This lane's share of the `want` greatest of the warp's 32 keys: the
 * want-th greatest, equal keys of different lanes counted apart. */
__device__ __forceinline__ uint32_t warp_nth(uint32_t key, int want) {
    uint32_t top = 0;
    for (int i = 0; i < want; i++) {
        top = __reduce_max_sync(0xffffffffu, key);
        const unsigned who = __ballot_sync(0xffffffffu, key == top);
        if ((threadIdx.x & 31) == __ffs(who) - 1)
            key = 0;
    }
    return top;
}

struct List {
    unsigned long long key[kListed];
    uint32_t least[kWarps];
    unsigned long long best[kWarps];
    int n;
};

/* Logits e0 .. e0 + kBeamEach - 1 (by thread and turn) of a chunk whose first
 * element lies `shift` elements behind a 16-byte boundary. */
template <typename T> struct Chunk {
    static constexpr int kPer = 16 / sizeof(T); /* elements of a load */
    static constexpr int kLoads = kBeamEach / kPer;
    /* element of the row that v[i] is */
    static __device__ __forceinline__ int64_t element(int64_t base, int i) {
        return base + (int64_t(i / kPer) * kBeamThreads + threadIdx.x) * kPer + i % kPer;
    }
    static __device__ __forceinline__ void load(const T *row, int64_t base, int vocab, float (&v)[kBeamEach]) {
#pragma unroll
        for (int k = 0; k < kLoads; k++) {
            const int64_t e = element(base, k * kPer);
            if (e >= 0 && e + kPer <= vocab) {
                const uint4 x = __ldcs(reinterpret_cast<const uint4 *>(row + e));
                const T *t = reinterpret_cast<const T *>(&x);
#pragma unroll
                for (int j = 0; j < kPer; j++)
                    v[k * kPer + j] = counted(to_float(t[j]));
            } else {
#pragma unroll
                for (int j = 0; j < kPer; j++)
                    v[k * kPer + j] = e + j >= 0 && e + j < vocab ? counted(to_float(row[e + j])) : -INFINITY;
            }
        }
    }
};

template <typename T>
__global__ void __launch_bounds__(kBeamThreads) chunk_kernel(const __grid_constant__ BeamSelect a) {
    __shared__ List list;
    __shared__ float tops[kWarps], sums[kWarps];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0)
        list.n = 0;
    begin_kernel();
    const int chunk = blockIdx.x;
    const int64_t r = blockIdx.y;
    if (a.finished && a.finished[r])
        return;
    const T *row = static_cast<const T *>(a.logits) + r * a.stride;
    const int shift = int((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
    const int64_t base = int64_t(chunk) * kBeamChunk - shift;
    float v[kBeamEach];
    Chunk<T>::load(row, base, a.vocab, v);

    float mine = v[0];
#pragma unroll
    for (int i = 1; i < kBeamEach; i++)
        mine = fmaxf(mine, v[i]);
    const float warp_top = warp_max(mine);
    /* the last chunk's first warps alone may have logits for all of their lanes */
    const int64_t there = (a.vocab - base) / (32 * Chunk<T>::kPer);
    const int full = there < kWarps ? int(there) : kWarps;
    const int want = full > 0 ? (a.n_out + full - 1) / full : 33;
    const uint32_t least = want > 32 ? 0u : warp < full ? warp_nth(ordered_bits(mine), want) : ~0u;
    if (lane == 0) {
        tops[warp] = warp_top;
        list.least[warp] = least;
    }
    __syncthreads();
    float top = tops[0];
    uint32_t edge = list.least[0];
#pragma unroll
    for (int w = 1; w < kWarps; w++) {
        top = fmaxf(top, tops[w]);
        edge = min(edge, list.least[w]);
    }
    const float from = top == -INFINITY ? 0.0f : top;
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < kBeamEach; i++)
        sum += exp2f((v[i] - from) * kLog2e);
    sum = warp_sum(sum);
    if (lane == 0)
        sums[warp] = sum;

    /* the logits that reach the edge, but not the places outside the row */
    const bool whole = base >= 0 && base + kBeamChunk <= a.vocab;
    if (ordered_bits(mine) >= edge)
#pragma unroll
        for (int i = 0; i < kBeamEach; i++)
            if (ordered_bits(v[i]) >= edge) {
                const int64_t e = Chunk<T>::element(base, i);
                if (whole || (e >= 0 && e < a.vocab)) {
                    const int at = atomicAdd(&list.n, 1);
                    if (at < kListed)
                        list.key[at] = argmax_key(v[i], uint32_t(e));
                }
            }
    __syncthreads();
    const int n = list.n;
    const int64_t part = r * a.chunks + chunk;
    unsigned long long *best = a.best + part * a.n_out;
    if (tid == 0) {
        float all = sums[0];
#pragma unroll
        for (int w = 1; w < kWarps; w++)
            all += sums[w];
        a.parts[part] = {top, all};
    }
    if (n <= kListed) {
        for (int i = tid; i < n; i += kBeamThreads) {
            const unsigned long long key = list.key[i];
            int rank = 0;
            for (int j = 0; j < n; j++)
                rank += list.key[j] > key;
            if (rank < a.n_out)
                best[rank] = key;
        }
        for (int i = n + tid; i < a.n_out; i += kBeamThreads)
            best[i] = 0;
        return;
    }
    /* equal logits: one after the other */
    unsigned long long last = ~0ull;
    for (int k = 0; k < a.n_out; k++) {
        unsigned long long key = 0;
#pragma unroll
        for (int i = 0; i < kBeamEach; i++) {
            const int64_t e = Chunk<T>::element(base, i);
            const unsigned long long x = argmax_key(v[i], uint32_t(e));
            if (e >= 0 && e < a.vocab && x < last && x > key)
                key = x;
        }
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) {
            const unsigned long long other = __shfl_xor_sync(0xffffffffu, key, x);
            key = other > key ? other : key;
        }
        if (lane == 0)
            list.best[warp] = key;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kWarps; w++)
            key = list.best[w] > key ? list.best[w] : key;
        if (tid == 0)
            best[k] = key;
        last = key;
        __syncthreads();
    }
}

/* ---- the choice among a request's chunks ------------------------------- */

/* An order-preserving map of a double (no NaN) to 64 bits, -0 folded onto +0,
 * and back. */
__device__ __forceinline__ unsigned long long ordered_double(double v) {
    const unsigned long long u = static_cast<unsigned long long>(__double_as_longlong(v == 0.0 ? 0.0 : v));
    return u >> 63 ? ~u : u | (1ull << 63);
}
__device__ __forceinline__ double double_of(unsigned long long bits) {
    return __longlong_as_double(static_cast<long long>(bits >> 63 ? bits & ~(1ull << 63) : ~bits));
}
__device__ __forceinline__ float float_of(uint32_t bits) {
    return __uint_as_float(bits & 0x80000000u ? bits & 0x7fffffffu : ~bits);
}

/* The greater score is first, then the lower place, beam * vocab + token. */
struct Candidate {
    unsigned long long score, place;
    __device__ __forceinline__ bool before(const Candidate &x) const {
        return score > x.score || (score == x.score && place < x.place);
    }
};

struct Choice {
    Candidate of[kListed], best[kWarps];
    uint32_t least[kWarps];
    int n;
};

struct Beam {
    double lse;
    float score;
    int ended;
};

/* Candidate i of a request whose beams begin at row0; false: there is none.
 * i counts (beam, chunk, rank). */
__device__ __forceinline__ bool candidate(const BeamSelect &a, const Beam *beams, int64_t row0, int i, Candidate &c) {
    const int per = a.chunks * a.n_out, b = i / per;
    const Beam beam = beams[b];
    if (beam.ended && i != b * per)
        return false;
    double score = beam.score;
    c.place = static_cast<unsigned long long>(b) * a.vocab;
    if (beam.ended) {
        c.place += a.eos;
    } else {
        const unsigned long long key = a.best[row0 * per + i];
        if (key == 0)
            return false;
        score += double(float_of(uint32_t(key >> 32))) - beam.lse;
        c.place += argmax_index(key);
    }
    c.score = ordered_double(score != score ? double(-INFINITY) : score);
    return true;
}

__device__ __forceinline__ void write_choice(const BeamSelect &a, const Beam *beams, int s, int k, const Candidate *c) {
    const int64_t to = int64_t(s) * a.n_out + k;
    const int beam = c ? int(c->place / a.vocab) : 0;
    const int64_t row = c ? int64_t(s) * a.beams + beam : -1;
    const int token = c ? int(c->place % a.vocab) : -1;
    a.out_scores[to] = c ? float(double_of(c->score)) : -INFINITY;
    a.out_rows[to] = int(row);
    a.out_tokens[to] = token;
    if (a.out_finished)
        a.out_finished[to] = c && (beams[beam].ended || token == a.eos);
}

__global__ void __launch_bounds__(kBeamThreads) join_kernel(const __grid_constant__ BeamSelect a) {
    /* [beams]; scores and finished are read once, their buffers may be the outputs */
    extern __shared__ Beam beams[];
    __shared__ Choice choice;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, s = blockIdx.x;
    if (tid == 0)
        choice.n = 0;
    begin_kernel();
    const int64_t row0 = int64_t(s) * a.beams;
    for (int b = warp; b < a.beams; b += kWarps) {
        const BeamPart *parts = a.parts + (row0 + b) * a.chunks;
        const bool ended = a.finished && a.finished[row0 + b];
        float top = -INFINITY;
        for (int c = lane; c < a.chunks && !ended; c += 32)
            top = fmaxf(top, parts[c].top);
        top = warp_max(top);
        double sum = 0.0;
        for (int c = lane; c < a.chunks && top != -INFINITY; c += 32)
            sum += parts[c].sum * exp(double(parts[c].top) - double(top));
#pragma unroll
        for (int x = 16; x > 0; x >>= 1)
            sum += __shfl_xor_sync(0xffffffffu, sum, x);
        if (lane == 0)
            beams[b] = {top == -INFINITY ? double(-INFINITY) : double(top) + log(sum), a.scores[row0 + b], ended};
    }
    __syncthreads();

    const int all = a.beams * a.chunks * a.n_out;
    uint32_t mine = 0; /* upper half of the best score */
    for (int i = tid; i < all; i += kBeamThreads) {
        Candidate c;
        if (candidate(a, beams, row0, i, c))
            mine = max(mine, uint32_t(c.score >> 32));
    }
    const uint32_t least = warp_nth(mine, (a.n_out + kWarps - 1) / kWarps);
    if (lane == 0)
        choice.least[warp] = least;
    __syncthreads();
    uint32_t edge = choice.least[0];
#pragma unroll
    for (int w = 1; w < kWarps; w++)
        edge = min(edge, choice.least[w]);
    if (mine >= edge)
        for (int i = tid; i < all; i += kBeamThreads) {
            Candidate c;
            if (candidate(a, beams, row0, i, c) && uint32_t(c.score >> 32) >= edge) {
                const int at = atomicAdd(&choice.n, 1);
                if (at < kListed)
                    choice.of[at] = c;
            }
        }
    __syncthreads();
    const int n = choice.n;
    if (n <= kListed) {
        for (int i = tid; i < n; i += kBeamThreads) {
            const Candidate c = choice.of[i];
            int rank = 0;
            for (int j = 0; j < n; j++)
                rank += choice.of[j].before(c);
            if (rank < a.n_out)
                write_choice(a, beams, s, rank, &c);
        }
        for (int i = n + tid; i < a.n_out; i += kBeamThreads)
            write_choice(a, beams, s, i, nullptr);
        return;
    }
    /* many equal scores: one after the other */
    Candidate last{~0ull, 0};
    bool any = true;
    for (int k = 0; k < a.n_out; k++) {
        Candidate best{0, ~0ull}; /* behind every candidate */
        for (int i = tid; i < all && any; i += kBeamThreads) {
            Candidate c;
            if (candidate(a, beams, row0, i, c) && (k == 0 || last.before(c)) && c.before(best))
                best = c;
        }
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) {
            const Candidate other{__shfl_xor_sync(0xffffffffu, best.score, x),
                                  __shfl_xor_sync(0xffffffffu, best.place, x)};
            if (other.before(best))
                best = other;
        }
        if (lane == 0)
            choice.best[warp] = best;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kWarps; w++)
            if (choice.best[w].before(best))
                best = choice.best[w];
        any = best.place != ~0ull;
        if (tid == 0)
            write_choice(a, beams, s, k, any ? &best : nullptr);
        last = best;
        __syncthreads();
    }
}

template <typename T> cudaError_t launch_chunks(const BeamSelect &a, cudaStream_t s) {
    return launch_kernel(chunk_kernel<T>, dim3(a.chunks, a.sequences * a.beams), kBeamThreads, 0, s, 1, a);
}

} // namespace

cudaError_t beam_select(const BeamSelect &a, cudaStream_t s) {
    const cudaError_t e = a.type == 0   ? launch_chunks<float>(a, s)
                          : a.type == 1 ? launch_chunks<__half>(a, s)
                                        : launch_chunks<__nv_bfloat16>(a, s);
    if (e != cudaSuccess)
        return e;
    return launch_kernel(join_kernel, dim3(a.sequences), kBeamThreads, a.beams * sizeof(Beam), s, 1, a);
}

} // namespace nut
