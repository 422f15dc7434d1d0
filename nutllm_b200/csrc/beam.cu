/* Beam search's choice over beams and vocabulary (nut_beam_select).
 *
 *   score(b, t) = scores[b] + logit[b][t] - log sum_u exp(logit[b][u])
 * The logits are read once, by warps that need no one else: each takes a run
 * of a row, 1,024 logits at a time (while the next ones are on their way to
 * shared memory), and keeps a maximum and a sum of exponentials for each lane
 * and a list in shared memory of what can be among the run's n_out greatest.
 * The first logits set an edge that n_out of them reach; from then on only what
 * is above it is listed, and a full list is reduced to its n_out greatest, the
 * last of which is the new edge.  Then a block for each request joins the runs' sums in fp64, turns what they listed
 * into scores and chooses among them: an edge from its threads' maxima, what
 * reaches it ranked by counting.
 *
 * Instructions bound the runs where there is much to read: 256 rows of 128,000
 * fp32 logits (123 MB without the ended beams') 33.8 us, 3.6 TB/s, 14.7
 * million warp instructions at 0.47 a cycle and scheduler.  The choice is a chain of
 * barriers and round trips, 9 to 12 us.  In a persistent grid whose last block
 * of a request chose, the requests' choices came one behind another.
 *
 * Sums: exponentials and a lane's sum in fp32, all beyond it in fp64.  Scores
 * are compared in fp64: a logit is fp32, and in an fp32 sum neighbours of
 * different beams would often round to a tie.
 */
#include <cfloat>
#include <cstdint>
#include <cuda_runtime.h>

#include "branch.h"
#include "paged.cuh"

namespace nut {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kEach = kBeamTile / 32; /* logits of a lane */
using Key = unsigned long long;       /* argmax_key(): the greater logit, then the lower token */

/* A logit as it counts: NaN as -infinity, +infinity as the greatest float. */
__device__ __forceinline__ float counted(float v) { return fminf(fmaxf(v, -INFINITY), FLT_MAX); }

/* 2^x, 0 below 2^-126. */
__device__ __forceinline__ float power2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}

/* The float of ordered_bits(). */
__device__ __forceinline__ float float_of(uint32_t bits) {
    return __uint_as_float(bits & 0x80000000u ? bits & 0x7fffffffu : ~bits);
}

/* The want-th greatest of the warp's 32 keys, equal ones counted apart. */
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

/* ---- a run of a row --------------------------------------------------- */

constexpr int kFull = 96;    /* keys of a warp's list; where there are more, they are reduced */
constexpr int kListed = 128; /* and room for one more of each lane */
constexpr int kRunWarps = 4;
static_assert(kListed >= kFull + 32 && kFull >= kBeamMostOut, "a logit of each lane at a time");

/* Leaves the `want` greatest of a warp's n keys, in descending order, and
 * returns how many there are. */
__device__ __noinline__ int reduce_list(Key *list, int n, int want) {
    const int lane = threadIdx.x & 31;
    constexpr int kOwn = kListed / 32;
    __syncwarp();
    if (n > 2 * want && want <= 32) {
        /* only those that reach the want-th of the lanes' maxima */
        Key own[kOwn], most = 0;
#pragma unroll
        for (int k = 0; k < kOwn; k++) {
            own[k] = k * 32 + lane < n ? list[k * 32 + lane] : 0;
            most = own[k] > most ? own[k] : most;
        }
        const uint32_t reach = warp_nth(uint32_t(most >> 32), want);
        int left = 0;
        __syncwarp();
#pragma unroll
        for (int k = 0; k < kOwn; k++) {
            const bool stays = own[k] != 0 && uint32_t(own[k] >> 32) >= reach;
            const unsigned who = __ballot_sync(0xffffffffu, stays);
            if (stays)
                list[left + __popc(who & ((1u << lane) - 1u))] = own[k];
            left += __popc(who);
        }
        n = left;
        __syncwarp();
    }
    if (lane < 8)
        list[n + lane] = 0; /* what follows reads 8 at a time */
    __syncwarp();
    Key own[kOwn];
    int rank[kOwn];
#pragma unroll
    for (int k = 0; k < kOwn; k++) {
        own[k] = k * 32 + lane < n ? list[k * 32 + lane] : 0;
        rank[k] = 0;
        if (k * 32 < n)
            for (int j = 0; j < n; j += 8)
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    const ulonglong2 x = *reinterpret_cast<const ulonglong2 *>(list + j + i);
                    rank[k] += (x.x > own[k]) + (x.y > own[k]);
                }
    }
    __syncwarp();
#pragma unroll
    for (int k = 0; k < kOwn; k++)
        if (k * 32 + lane < n && rank[k] < want)
            list[rank[k]] = own[k];
    __syncwarp();
    return min(n, want);
}

template <typename T>
__global__ void __launch_bounds__(kRunWarps * 32) runs_kernel(const __grid_constant__ BeamSelect a) {
    constexpr int kPer = 16 / sizeof(T); /* elements of a load */
    __shared__ alignas(16) Key lists[kRunWarps][kListed + 8];
    begin_kernel();
    const int lane = threadIdx.x & 31;
    const int part = int(blockIdx.x) * kRunWarps + int(threadIdx.x >> 5), row = part / a.runs;
    if (row >= a.sequences * a.beams || (a.finished && a.finished[row]))
        return;
    Key *list = lists[threadIdx.x >> 5];
    const T *logits = static_cast<const T *>(a.logits) + row * a.stride;
    /* tiles begin at 16-byte boundaries, the first up to 15 bytes before the row */
    const int shift = int((reinterpret_cast<uintptr_t>(logits) & 15) / sizeof(T));
    int base = (part - row * a.runs) * a.run_tiles * kBeamTile - shift;
    const int end = min(base + a.run_tiles * kBeamTile, a.vocab);
    constexpr int kLoads = kEach / kPer;
    extern __shared__ uint4 stages[];
    uint4 *stage = stages + (threadIdx.x >> 5) * (2 * kLoads * 32); /* of two tiles; place i * 32 + lane */
    const auto whole = [&](int from) { return from >= 0 && from + kBeamTile <= a.vocab; };
    const auto begin = [&](int from, uint4 *to) {
        if (from < end && whole(from))
#pragma unroll
            for (int i = 0; i < kLoads; i++)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(
                                 uint32_t(__cvta_generic_to_shared(to + i * 32 + lane))),
                             "l"(logits + from + (i * 32 + lane) * kPer)
                             : "memory");
        asm volatile("cp.async.commit_group;\n" ::: "memory");
    };
    begin(base, stage);
    float top = -INFINITY, sum = 0.0f; /* this lane's */
    Key edge = 0;                      /* what is listed is greater */
    int n = 0;
    for (int turn = 0; base < end; base += kBeamTile, turn ^= 1) {
        uint4 *now = stage + turn * (kLoads * 32);
        begin(base + kBeamTile, stage + (turn ^ 1) * (kLoads * 32));
        asm volatile("cp.async.wait_group 1;\n" ::: "memory");
        /* a lane reads what it copied: element i is that of place at(i) */
        float v[kEach];
        const auto at = [&](int i) { return base + (i / kPer * 32 + lane) * kPer + i % kPer; };
        if (!whole(base)) /* the row's ends */
#pragma unroll 1
            for (int i = 0; i < kEach; i++) {
                const int e = at(i);
                reinterpret_cast<T *>(now + i / kPer * 32 + lane)[i % kPer] =
                    e >= 0 && e < a.vocab ? logits[e] : output_of<T>(-INFINITY);
            }
#pragma unroll
        for (int i = 0; i < kLoads; i++) {
            const uint4 x = now[i * 32 + lane];
#pragma unroll
            for (int j = 0; j < kPer; j++)
                v[i * kPer + j] = to_float(reinterpret_cast<const T *>(&x)[j]);
        }
        float most = -INFINITY, next = -INFINITY; /* of every other load; NaN is never the greater */
#pragma unroll
        for (int i = 0; i < kEach; i++)
            if (i / kPer % 2 == 0)
                most = fmaxf(most, v[i]);
            else
                next = fmaxf(next, v[i]);
        if (fmaxf(most, next) == INFINITY) { /* seldom */
#pragma unroll
            for (int i = 0; i < kEach; i++)
                v[i] = counted(v[i]);
            most = fminf(most, FLT_MAX);
            next = fminf(next, FLT_MAX);
        }
        if (edge == 0) {
            /* n_out of these reach the n_out-th of the lanes' maxima, or the least of the
             * two that each lane has; the key below it is the edge */
            const uint32_t reach = a.n_out <= 32 ? warp_nth(ordered_bits(fmaxf(most, next)), a.n_out)
                                                 : __reduce_min_sync(0xffffffffu, ordered_bits(fminf(most, next)));
            edge = (Key(reach) << 32) - 1;
        }
        most = fmaxf(most, next);
        if (most > top) {
            sum *= power2((top - most) * kLog2e);
            top = most;
        }
        const float from = top == -INFINITY ? 0.0f : top;
        Two more2 = two_of(0.0f, 0.0f);
        const Two less = two_of(-from, -from), scale = two_of(kLog2e, kLog2e);
#pragma unroll
        for (int i = 0; i < kEach; i += 2) { /* (v - from) log2 e */
            Two x = two_of(v[i], v[i + 1]);
            asm("add.rn.f32x2 %0, %0, %1;\n" : "+l"(x) : "l"(less));
            asm("mul.rn.f32x2 %0, %0, %1;\n" : "+l"(x) : "l"(scale));
            const float2 z = parts_of(x);
            asm("add.rn.f32x2 %0, %0, %1;\n" : "+l"(more2) : "l"(two_of(power2(z.x), power2(z.y))));
        }
        const float2 parts = parts_of(more2);
        float more = parts.x + parts.y;
        if (more != more) { /* there is a NaN among them: again, without it */
            more = 0.0f;
#pragma unroll 1
            for (int i = 0; i < kEach; i++)
                more += power2((counted(to_float(reinterpret_cast<const T *>(now + i / kPer * 32 + lane)[i % kPer])) - from) * kLog2e);
        }
        sum += more;

        /* what is above the edge, by value first: its key is that of an earlier token, which
         * wins a tie, or the one below n_out equal ones */
        const uint32_t edge_bits = uint32_t(edge >> 32), lowest = 0x007fffffu; /* of -infinity */
        const bool any = edge_bits < lowest || ordered_bits(most) > edge_bits;
        if (!__any_sync(0xffffffffu, any))
            continue;
        uint32_t hits = 0;
        if (edge_bits < lowest) {
            hits = ~0u; /* every logit, NaN too, which counts as -infinity */
        } else if (any) {
            /* (below +0, which -0 counts as too, comes the least negative number) */
            const float edge_value = float_of(edge_bits == 0x7fffffffu ? 0x7ffffffeu : edge_bits);
#pragma unroll
            for (int i = 0; i < kEach; i++)
                hits |= uint32_t(v[i] > edge_value) << i;
        }
        /* a logit of each lane at a time, from where it lies: registers have no index */
        while (__any_sync(0xffffffffu, hits != 0)) {
            Key key = 0;
            if (hits != 0) {
                const int i = __ffs(hits) - 1, e = at(i);
                hits &= hits - 1;
                if (e >= 0 && e < a.vocab)
                    key = argmax_key(counted(to_float(reinterpret_cast<const T *>(now + i / kPer * 32 + lane)[i % kPer])), uint32_t(e));
            }
            const bool hit = key > edge;
            const unsigned who = __ballot_sync(0xffffffffu, hit);
            if (hit)
                list[n + __popc(who & ((1u << lane) - 1u))] = key;
            n += __popc(who);
            if (n > kFull) {
                n = reduce_list(list, n, a.n_out);
                edge = list[n - 1]; /* n_out of them are left */
            }
        }
    }
    n = reduce_list(list, n, a.n_out);
    Key *best = a.best + int64_t(part) * a.n_out;
    for (int i = lane; i < a.n_out; i += 32)
        best[i] = i < n ? list[i] : 0;
    const float most = warp_max(top);
    const float share = sum == 0.0f ? 0.0f : sum * power2((top - most) * kLog2e);
    double total = share;
#pragma unroll
    for (int x = 16; x > 0; x >>= 1)
        total += __shfl_xor_sync(0xffffffffu, total, x);
    if (lane == 0)
        a.parts[part] = {total, most};
}

/* ---- the choice among a request's runs ---------------------------------- */

/* An order-preserving map of a double (no NaN) to 64 bits, -0 folded onto +0,
 * and back. */
__device__ __forceinline__ unsigned long long ordered_double(double v) {
    const unsigned long long u = static_cast<unsigned long long>(__double_as_longlong(v == 0.0 ? 0.0 : v));
    return u >> 63 ? ~u : u | (1ull << 63);
}
__device__ __forceinline__ double double_of(unsigned long long bits) {
    return __longlong_as_double(static_cast<long long>(bits >> 63 ? bits & ~(1ull << 63) : ~bits));
}

/* The greater score is first, then the lower place: beam, then token. */
struct Candidate {
    unsigned long long score, place;
    __device__ __forceinline__ bool before(const Candidate &x) const {
        return score > x.score || (score == x.score && place < x.place);
    }
};

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kMany = 512; /* candidates that are ranked by counting */

struct Choice {
    Candidate of[kMany], best[kWarps];
    int n;
};

struct Beam {
    double lse;
    float score;
    int ended;
};

/* Entry `rank` of what run `run` of beam b listed, as a candidate; false: there is none.
 * An ended beam has one.  All tokens of a beam whose score is -infinity (or NaN)
 * tie, and the lowest are first: those, not the greatest logits that its runs
 * listed. */
__device__ __forceinline__ bool candidate(const BeamSelect &a, const Beam *beams, int b, int run, int rank, Key key,
                                          Candidate &c) {
    const Beam beam = beams[b];
    const bool none = !(beam.score > -INFINITY);
    if (beam.ended ? run != 0 || rank != 0 : none ? run != 0 || rank >= a.vocab : key == 0)
        return false;
    double score = none ? double(-INFINITY) : double(beam.score);
    c.place = static_cast<unsigned long long>(b) << 32;
    if (beam.ended) {
        c.place += a.eos;
    } else if (none) {
        c.place += rank;
    } else {
        score += double(float_of(uint32_t(key >> 32))) - beam.lse;
        c.place += argmax_index(key);
    }
    c.score = ordered_double(score != score ? double(-INFINITY) : score);
    return true;
}

__device__ __forceinline__ void write_choice(const BeamSelect &a, const Beam *beams, int s, int k, const Candidate *c) {
    const int64_t to = int64_t(s) * a.n_out + k;
    const int beam = c ? int(c->place >> 32) : 0;
    const int64_t row = c ? int64_t(s) * a.beams + beam : -1;
    const int token = c ? int(c->place) : -1;
    a.out_scores[to] = c ? float(double_of(c->score)) : -INFINITY;
    a.out_rows[to] = int(row);
    a.out_tokens[to] = token;
    if (a.out_finished)
        a.out_finished[to] = c && (beams[beam].ended || token == a.eos);
}

/* A key that at least `want` of the block's reach, and few more. */
__device__ __forceinline__ uint32_t block_edge(uint32_t key, int want) {
    uint32_t lo = 0, hi = ~0u; /* `want` reach lo, fewer reach hi */
    while (hi - lo > 1) {
        const uint32_t mid = lo + (hi - lo) / 2;
        const int many = __syncthreads_count(key >= mid);
        if (many >= want) {
            lo = mid;
            if (many <= want + want / 4)
                break;
        } else {
            hi = mid;
        }
    }
    return lo;
}

/* The block's candidates: f(candidate) for each.  A list's entries lie in
 * neighbouring lanes, kBatch lists of a lane are in flight. */
template <typename F>
__device__ __forceinline__ void for_candidates(const BeamSelect &a, const Beam *beams, int64_t row0, F &&f) {
    const int across = a.n_out > 16 ? 32 : a.n_out > 8 ? 16 : a.n_out > 4 ? 8 : 4; /* lanes of a list */
    const int lists = a.beams * a.runs, step = kThreads / across, place = threadIdx.x & (across - 1);
    constexpr int kBatch = 4;
    for (int l0 = threadIdx.x / across; l0 < lists; l0 += kBatch * step)
        for (int rank = place; rank < a.n_out; rank += across) {
            Key keys[kBatch];
#pragma unroll
            for (int k = 0; k < kBatch; k++)
                keys[k] = l0 + k * step < lists ? a.best[(row0 * a.runs + l0 + k * step) * a.n_out + rank] : 0;
#pragma unroll
            for (int k = 0; k < kBatch; k++) {
                const int list = l0 + k * step, b = list / a.runs;
                Candidate c;
                if (list < lists && candidate(a, beams, b, list - b * a.runs, rank, keys[k], c))
                    f(c);
            }
        }
}

__global__ void __launch_bounds__(kThreads) choose_kernel(const __grid_constant__ BeamSelect a) {
    /* [beams]; scores and finished are read once, their buffers may be the outputs */
    extern __shared__ Beam beams[];
    __shared__ Choice choice;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, s = blockIdx.x;
    if (tid == 0)
        choice.n = 0;
    begin_kernel();
    const int64_t row0 = int64_t(s) * a.beams;
    for (int b = warp; b < a.beams; b += kWarps) {
        const BeamPart *parts = a.parts + (row0 + b) * a.runs;
        const bool ended = a.finished && a.finished[row0 + b];
        const float score = a.scores[row0 + b];
        float top = -INFINITY;
        double sum = 0.0;
        for (int c = lane; c < a.runs && !ended; c += 32) {
            const BeamPart x = parts[c];
            if (x.top > top) {
                sum *= top == -INFINITY ? 0.0 : exp(double(top) - double(x.top));
                top = x.top;
            }
            if (x.top != -INFINITY)
                sum += x.sum * exp(double(x.top) - double(top));
        }
        const float most = warp_max(top);
        if (top != most)
            sum *= top == -INFINITY ? 0.0 : exp(double(top) - double(most));
#pragma unroll
        for (int x = 16; x > 0; x >>= 1)
            sum += __shfl_xor_sync(0xffffffffu, sum, x);
        if (lane == 0)
            beams[b] = {most == -INFINITY ? double(-INFINITY) : double(most) + log(sum), score, ended};
    }
    __syncthreads();

    uint32_t mine = 0; /* upper half of the best score */
    for_candidates(a, beams, row0, [&](const Candidate &c) { mine = max(mine, uint32_t(c.score >> 32)); });
    const uint32_t edge = block_edge(mine, a.n_out);
    if (mine >= edge)
        for_candidates(a, beams, row0, [&](const Candidate &c) {
            if (uint32_t(c.score >> 32) >= edge) {
                const int at = atomicAdd(&choice.n, 1);
                if (at < kMany)
                    choice.of[at] = c;
            }
        });
    __syncthreads();
    const int n = choice.n;
    if (n <= kMany) {
        for (int i = tid; i < n; i += kThreads) {
            const Candidate c = choice.of[i];
            int rank = 0;
#pragma unroll 4
            for (int j = 0; j < n; j++)
                rank += choice.of[j].before(c);
            if (rank < a.n_out)
                write_choice(a, beams, s, rank, &c);
        }
        for (int i = n + tid; i < a.n_out; i += kThreads)
            write_choice(a, beams, s, i, nullptr);
        return;
    }
    /* many equal scores: the best one after the other, each thread with the best of
     * its own at hand */
    Candidate last{~0ull, 0}, own{0, ~0ull}; /* ~0: behind every candidate */
    bool stale = true;
    for (int k = 0; k < a.n_out; k++) {
        if (stale) {
            own = {0, ~0ull};
            for_candidates(a, beams, row0, [&](const Candidate &c) {
                if ((k == 0 || last.before(c)) && c.before(own))
                    own = c;
            });
        }
        Candidate best = own;
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
        const bool any = best.place != ~0ull;
        if (tid == 0)
            write_choice(a, beams, s, k, any ? &best : nullptr);
        stale = any && best.place == own.place;
        last = best;
        __syncthreads();
    }
}

template <typename T> cudaError_t launch_runs(const BeamSelect &a, cudaStream_t s) {
    const int parts = a.sequences * a.beams * a.runs;
    return launch_kernel(runs_kernel<T>, dim3((parts + kRunWarps - 1) / kRunWarps), kRunWarps * 32,
                         kRunWarps * 2 * kBeamTile * sizeof(T), s, 1, a);
}

} // namespace

cudaError_t beam_select(const BeamSelect &a, cudaStream_t s) {
    const cudaError_t e = a.type == 0   ? launch_runs<float>(a, s)
                          : a.type == 1 ? launch_runs<__half>(a, s)
                                        : launch_runs<__nv_bfloat16>(a, s);
    if (e != cudaSuccess)
        return e;
    return launch_kernel(choose_kernel, dim3(a.sequences), kThreads, a.beams * sizeof(Beam), s, 1, a);
}

} // namespace nut
