/* Attention of one token per row over the paged KV cache
 * (nut_paged_attention).
 *
 *   z_t = scale q . k_t,  m = max z,  l = sum exp(z_t - m),
 *   out = sum exp(z_t - m) v_t / l,   lse = m + log l
 * in one pass over the keys and values with a running maximum and sum.
 *
 * Work.  A row, a kv head and up to 8 of its query heads are an item; an
 * item's slots are cut into tiles, and all tiles of all items form one line
 * that is cut evenly among the CTAs whatever the lengths.  An item that lies
 * in one CTA is finished there.  Of one that spans several, each leaves its
 * unnormalised output, maximum and sum, and the last to arrive joins them
 * in order of their slots, so results do not depend on timing.
 *
 * HBM bounds it: 62 sequences of up to 4,096 slots, 32/8 heads of 128, bf16,
 * are 545 MB and take 100 us (5.45 TB/s, 83 % of a measured copy; 4 us pass
 * before the first keys arrive and 5 at the end to join).  Where the pages
 * come out of L2 (256 queries of one prompt, 2.1 GB) it is the latency of a
 * warp's own products and softmax, 128 us; dense rows of a prompt re-read the
 * cache for every row (512 rows behind 8,192 slots: 1.3 ms).  Calls of a few tiles are a chain
 * of round trips: 37 slots take 6.7 us.
 */
#include <cstdint>
#include <type_traits>
#include <cuda_runtime.h>

#include "paged.cuh"
#include "stream.cuh"

namespace nut {
namespace {

constexpr int kChunk = 16; /* slots a warp takes at a time */
constexpr int kRows = 8;   /* query heads of an item */
constexpr int kBlock = kChunk * 128; /* a chunk's 128-byte columns, in the 128-byte swizzle */
/* What an item costs besides its tiles, in tiles: with 0, 1, 2 and 3 a batch
 * whose shares hold 1 to 20 items took 147, 108, 101 and 100 us. */
constexpr int kItemCost = 3;
/* log2 by which a logit may pass the maximum in use: with kLift, which may
 * round to 8 beside a maximum of 2^24 or more, 2^15 at most */
constexpr float kSlack = 7.0f;
constexpr uint64_t kPagedWaitNs = 2000000000ull;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

/* One box of the pool to shared memory: from column x of 128-byte column b,
 * the map's slots from y, kv head h, page w; arrives on `bar`. */
__device__ __forceinline__ void copy_box(uint32_t to, const CUtensorMap *map, int x, int y, int b, int h, int w,
                                         uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
                 "[%0], [%1, {%3, %4, %5, %6, %7}], [%2];\n" ::"r"(to),
                 "l"(map), "r"(bar), "r"(x), "r"(y), "r"(b), "r"(h), "r"(w)
                 : "memory");
}
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory"); }
__device__ __forceinline__ void fence_proxy_async() { asm volatile("fence.proxy.async;\n" ::: "memory"); }

/* Waits for a stage without sleeping; false after kPagedWaitNs. */
__device__ __forceinline__ bool stage_wait(uint64_t *bar, uint32_t parity) {
    uint64_t start = 0;
    for (int i = 0;; i++) {
        if (mbar_try_wait(bar, parity))
            return true;
        if ((i & 63) == 63) {
            const uint64_t now = global_ns();
            if (start == 0)
                start = now;
            else if (now - start > kPagedWaitNs)
                return false;
        }
    }
}

__device__ __forceinline__ void load_matrices(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(at)
                 : "memory");
}
__device__ __forceinline__ void load_matrices_t(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(at)
                 : "memory");
}

template <typename T> struct Pair;
template <> struct Pair<__half> {
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
    static __device__ __forceinline__ float2 unpack(uint32_t v) {
        return __half22float2(*reinterpret_cast<const __half2 *>(&v));
    }
    static __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                               uint32_t a3, uint32_t b0, uint32_t b1) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, "
                     "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};\n"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    }
};
template <> struct Pair<__nv_bfloat16> {
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
    static __device__ __forceinline__ float2 unpack(uint32_t v) {
        return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&v));
    }
    static __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                               uint32_t a3, uint32_t b0, uint32_t b1) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, "
                     "{%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};\n"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    }
};

/* What is left of x, y after the 16-bit pair `taken` is taken away. */
template <typename T> __device__ __forceinline__ float2 left_of(float x, float y, uint32_t taken) {
    const float2 f = Pair<T>::unpack(taken);
    return make_float2(x - f.x, y - f.y);
}

/* hi + rest, but an infinite hi as it is: the lower terms of a product with
 * an infinity are infinities of any sign. */
__device__ __forceinline__ float plus_terms(float hi, float rest) {
    return fabsf(hi) == INFINITY ? hi : hi + rest;
}

/* ---- 16-bit caches: mma.sync m16n8k16 ------------------------------- *
 *
 * Of the 16 rows of an A operand only 8 can be different query heads that
 * share the keys (8 is Llama's largest group), so rows 8-15 carry what the
 * 16-bit rounding of rows 0-7 left out: a query is hi + lo, and c of row g
 * plus c of row g + 8, which lie in the same thread, is the fp32 logit at no
 * further cost.  The weights of the second product are split the same way.
 * fp16's two terms hold 22 bits (fp32 queries are first scaled by a power
 * of two into its range), bf16's two hold 16, less than a bf16 output's
 * rounding loses; with fp32 rows a third bf16 term goes through a second mma.
 * fp16 ends at 2^-24, below which what many small weights add up to would be
 * lost beside one great one (a quarter of an output made of 2,047 weights
 * 18 nats below the greatest).  So its weights are 2^kLift times as great, at
 * most 2^15 with kSlack, and their second terms, at most 2^4, kLow times that,
 * which the accumulators of rows 8-15, theirs alone, undo at the end: a weight
 * is within 2^-22 of itself or 2^-43 of the greatest. */
template <typename T, typename R, int DP_> struct Halves {
    static constexpr int DP = DP_, kWarps = 4;
    static constexpr bool kThird = std::is_same<T, __nv_bfloat16>::value && std::is_same<R, float>::value;
    static constexpr bool kScaled = std::is_same<T, __half>::value && std::is_same<R, float>::value;
    static constexpr bool kSplitQ = std::is_same<R, float>::value;
    static constexpr float kLift = std::is_same<T, __half>::value ? 7.0f : 0.0f; /* log2 */
    static constexpr float kLow = std::is_same<T, __half>::value ? 2048.0f : 1.0f;
    static constexpr int kMaxPerSm = DP >= 128 && kThird ? 2 : 3; /* by registers */
    static constexpr int kBlocks = (DP * 2 + 127) / 128; /* 128-byte columns of a row */
    static constexpr int kStageBytes = 2 * kBlocks * kBlock;
    static constexpr int kSteps = DP / 16;
    using Cache = T;

    uint32_t q[kSteps][kSplitQ ? 4 : 2], q3[kThird ? kSteps : 1][2];
    float o[DP / 8][4];
    float m, l, unit; /* running maximum (log2), this lane's share of the sum, logit unit */

    __device__ __forceinline__ void begin(const PagedAttention &a, const void *query, int heads,
                                          float *) {
        const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, D = a.p.head_dim;
        const R *x = static_cast<const R *>(query) + int64_t(g) * D;
        float top = 0.0f;
        if (kScaled && g < heads)
            for (int d = 2 * t; d < D; d += 8)
                top = fmaxf(top, fmaxf(fabsf(to_float(x[d])), fabsf(to_float(x[d + 1]))));
        float gain = 1.0f;
        unit = a.scale * kLog2e;
        if (kScaled) {
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            /* greatest |q| to [2^10, 2^11) */
            const int e = int(__float_as_uint(top) >> 23);
            if (e > 0 && e < 255) {
                const int field = min(264 - e, 253);
                gain = __uint_as_float(uint32_t(field) << 23);
                unit *= __uint_as_float(uint32_t(254 - field) << 23);
            }
        }
#pragma unroll
        for (int s = 0; s < kSteps; s++)
#pragma unroll
            for (int half = 0; half < 2; half++) {
                const int d = s * 16 + half * 8 + 2 * t;
                float v0 = 0.0f, v1 = 0.0f;
                if (g < heads && d < D) {
                    v0 = to_float(x[d]) * gain;
                    v1 = to_float(x[d + 1]) * gain;
                }
                const uint32_t hi = Pair<T>::pack(v0, v1);
                if constexpr (kSplitQ) {
                    const float2 r = left_of<T>(v0, v1, hi);
                    const uint32_t lo = Pair<T>::pack(r.x, r.y);
                    q[s][2 * half] = hi;
                    q[s][2 * half + 1] = lo;
                    if constexpr (kThird) {
                        const float2 r3 = left_of<T>(r.x, r.y, lo);
                        q3[s][half] = Pair<T>::pack(r3.x, r3.y);
                    }
                } else {
                    q[s][half] = hi;
                }
            }
        m = -INFINITY;
        l = 0.0f;
#pragma unroll
        for (int n = 0; n < DP / 8; n++)
            o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.0f;
    }

    /* 16 slots from the stage at `at`; bit t of `valid` says whether slot t
     * counts.  z (if not NULL) receives their log2 logits, [heads][stride]. */
    __device__ __forceinline__ void step(uint32_t at, uint32_t valid, float *, float *z, int stride,
                                         int heads) {
        const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
        float c[2][2][4], c3[2][4];
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int j = 0; j < 4; j++)
                c[0][i][j] = c[1][i][j] = c3[i][j] = 0.0f;
        /* 16-byte piece c of row r lies at piece c ^ (r & 7) of its 128 bytes */
        const uint32_t krow = at + ((lane >> 4) * 8 + (lane & 7)) * 128, kx = (((lane >> 3) & 1) ^ (lane & 7)) * 16;
#pragma unroll
        for (int s = 0; s < kSteps; s++) {
            uint32_t b[4];
            load_matrices(b, krow + (s / 4) * kBlock + (kx ^ ((s & 3) * 32)));
            if constexpr (kSplitQ) {
                Pair<T>::mma(c[s & 1][0], q[s][0], q[s][1], q[s][2], q[s][3], b[0], b[1]);
                Pair<T>::mma(c[s & 1][1], q[s][0], q[s][1], q[s][2], q[s][3], b[2], b[3]);
                if constexpr (kThird) {
                    Pair<T>::mma(c3[0], q3[s][0], 0u, q3[s][1], 0u, b[0], b[1]);
                    Pair<T>::mma(c3[1], q3[s][0], 0u, q3[s][1], 0u, b[2], b[3]);
                }
            } else {
                Pair<T>::mma(c[s & 1][0], q[s][0], 0u, q[s][1], 0u, b[0], b[1]);
                Pair<T>::mma(c[s & 1][1], q[s][0], 0u, q[s][1], 0u, b[2], b[3]);
            }
        }
        /* logits of head g, slots 8 i + 2 t + j, in units of log 2 */
        float s2[2][2], top = -INFINITY;
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
                float v = c[0][i][j] + c[1][i][j];
                if constexpr (kSplitQ)
                    v = plus_terms(v, c[0][i][2 + j] + c[1][i][2 + j] + c3[i][j]);
                v *= unit;
                if (valid != 0xffffu && !((valid >> (8 * i + 2 * t + j)) & 1))
                    v = -INFINITY;
                s2[i][j] = v;
                top = fmaxf(top, v);
            }
        if (z != nullptr && g < heads)
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int j = 0; j < 2; j++)
                    if ((valid >> (8 * i + 2 * t + j)) & 1)
                        z[int64_t(g) * stride + 8 * i + 2 * t + j] = s2[i][j];
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        /* the maximum in use may lag behind by kSlack (the difference is exact
         * where it matters): outputs are rarely rescaled */
        const float next = top - m > kSlack || m == -INFINITY ? fmaxf(m, top) : m;
        if (__any_sync(0xffffffffu, next != m)) {
            const float keep = m == next ? 1.0f : exp2f(m - next);
            l *= keep;
#pragma unroll
            for (int n = 0; n < DP / 8; n++) {
                o[n][0] *= keep;
                o[n][1] *= keep;
                o[n][2] *= keep;
                o[n][3] *= keep;
            }
            m = next;
        }
        const float base = m == -INFINITY ? 0.0f : m - kLift;
        uint32_t hi[2], lo[2], p3[2], tiny[2];
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const float w0 = exp2f(s2[i][0] - base), w1 = exp2f(s2[i][1] - base);
            l += w0 + w1;
            hi[i] = Pair<T>::pack(w0, w1);
            const float2 r = left_of<T>(w0, w1, hi[i]);
            lo[i] = Pair<T>::pack(r.x * kLow, r.y * kLow);
            if constexpr (kThird) {
                const float2 r3 = left_of<T>(r.x, r.y, lo[i]);
                p3[i] = Pair<T>::pack(r3.x, r3.y);
                const __nv_bfloat162 t = __hmul2(*reinterpret_cast<const __nv_bfloat162 *>(&hi[i]),
                                                 __float2bfloat162_rn(0x1p-40f));
                tiny[i] = *reinterpret_cast<const uint32_t *>(&t);
            }
        }
        const uint32_t vrow = at + kBlocks * kBlock + (lane & 15) * 128, vx = ((lane >> 4) ^ (lane & 7)) * 16;
#pragma unroll
        for (int n = 0; n < DP / 16; n++) {
            uint32_t b[4];
            load_matrices_t(b, vrow + (n / 4) * kBlock + (vx ^ ((n & 3) * 32)));
            Pair<T>::mma(o[2 * n], hi[0], lo[0], hi[1], lo[1], b[0], b[1]);
            Pair<T>::mma(o[2 * n + 1], hi[0], lo[0], hi[1], lo[1], b[2], b[3]);
            if constexpr (kThird) {
                /* into the rows of the second terms; the first ones get 2^-40
                 * of their weight, which changes nothing, but where 0 would
                 * make an infinite value NaN */
                Pair<T>::mma(o[2 * n], tiny[0], p3[0], tiny[1], p3[1], b[0], b[1]);
                Pair<T>::mma(o[2 * n + 1], tiny[0], p3[0], tiny[1], p3[1], b[2], b[3]);
            }
        }
    }

    /* This warp's maxima, kLift below the real ones, and sums of the 8 heads. */
    __device__ __forceinline__ void statistics(float *maxima, float *sums) {
        const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        if (t == 0) {
            maxima[g] = m - kLift;
            sums[g] = l;
        }
    }
    /* Its output, times factor[head], to out [8][DP], or added there. */
    template <bool kAdd> __device__ __forceinline__ void output(float *out, const float *factor) {
        const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
        const float f = factor[g];
#pragma unroll
        for (int n = 0; n < DP / 8; n++) {
            float2 *to = reinterpret_cast<float2 *>(out + g * DP + n * 8 + 2 * t);
            float2 v = make_float2(0.0f, 0.0f);
            if (f != 0.0f)
                v = make_float2(plus_terms(o[n][0], o[n][2] * (1.0f / kLow)) * f,
                                plus_terms(o[n][1], o[n][3] * (1.0f / kLow)) * f);
            if (kAdd)
                v = make_float2(v.x + to->x, v.y + to->y);
            *to = v;
        }
    }
};

/* ---- fp32 caches: FFMA ---------------------------------------------- *
 *
 * Logits: lane (slot, half) takes half of the dims of one of 16 slots for
 * all query heads (queries broadcast from shared memory); the halves meet
 * with one exchange, after which half h keeps heads h NQ/2 ...  Context: a
 * lane owns 4 dims, or with fewer than 128 dims 4 dims of a share of the
 * slots, for all heads. */
template <int NQ, int DP_> struct Wide {
    static constexpr int DP = DP_, kWarps = DP > 128 ? 2 : 4, kMaxPerSm = 3;
    static constexpr int kBlocks = DP / 32; /* 128-byte columns of a row */
    static constexpr int kStageBytes = 2 * kBlocks * kBlock;
    static constexpr int kOwn = NQ >= 2 ? NQ / 2 : 1; /* heads a lane does the softmax of */
    static constexpr int kQuads = DP / 4;             /* 4-dim pieces of a row */
    static constexpr int kLanes = kQuads < 32 ? (kQuads >= 16 ? 16 : 8) : 32; /* lanes across a row */
    static constexpr int kPieces = (kQuads + kLanes - 1) / kLanes;
    static constexpr int kShares = 32 / kLanes; /* lanes that share a piece, over slots */
    using Cache = float;

    float o[NQ][kPieces][4];
    float m[kOwn], l[kOwn], unit;

    /* scratch: queries [NQ][DP], then per slot weights [16][NQ], then keep [NQ] */
    static constexpr int kScratch = NQ * DP + kChunk * NQ + NQ + 3;

    __device__ __forceinline__ void begin(const PagedAttention &a, const void *query, int heads,
                                          float *scratch) {
        const int lane = threadIdx.x & 31, D = a.p.head_dim;
        const float *x = static_cast<const float *>(query);
        __syncwarp();
        for (int i = lane; i < NQ * DP; i += 32) {
            const int g = i / DP, d = i % DP;
            scratch[i] = g < heads && d < D ? x[int64_t(g) * D + d] : 0.0f;
        }
        __syncwarp();
        unit = a.scale * kLog2e;
#pragma unroll
        for (int g = 0; g < kOwn; g++) {
            m[g] = -INFINITY;
            l[g] = 0.0f;
        }
#pragma unroll
        for (int g = 0; g < NQ; g++)
#pragma unroll
            for (int n = 0; n < kPieces; n++)
#pragma unroll
                for (int j = 0; j < 4; j++)
                    o[g][n][j] = 0.0f;
    }

    __device__ __forceinline__ void step(uint32_t at, uint32_t valid, float *scratch, float *z,
                                         int stride, int heads) {
        const int lane = threadIdx.x & 31, slot = lane & 15, half = lane >> 4;
        const char *stage = static_cast<const char *>(__cvta_shared_to_generic(at));
        float s[NQ];
#pragma unroll
        for (int g = 0; g < NQ; g++)
            s[g] = 0.0f;
        /* 16-byte piece c of row r lies at piece c ^ (r & 7) of its 128 bytes */
        const char *krow = stage + slot * 128;
#pragma unroll 4
        for (int d = 0; d < DP / 2; d += 4) {
            const int piece = half * (DP / 8) + d / 4;
            const float4 k = *reinterpret_cast<const float4 *>(krow + (piece >> 3) * kBlock +
                                                               (((piece & 7) ^ (slot & 7)) << 4));
#pragma unroll
            for (int g = 0; g < NQ; g++) {
                const float4 x = *reinterpret_cast<const float4 *>(scratch + g * DP + half * (DP / 2) + d);
                s[g] = fmaf(x.x, k.x, s[g]);
                s[g] = fmaf(x.y, k.y, s[g]);
                s[g] = fmaf(x.z, k.z, s[g]);
                s[g] = fmaf(x.w, k.w, s[g]);
            }
        }
        float own[kOwn];
        if constexpr (NQ == 1) {
            own[0] = s[0] + __shfl_xor_sync(0xffffffffu, s[0], 16);
        } else {
#pragma unroll
            for (int g = 0; g < kOwn; g++) {
                const float give = half ? s[g] : s[g + kOwn], mine = half ? s[g + kOwn] : s[g];
                own[g] = mine + __shfl_xor_sync(0xffffffffu, give, 16);
            }
        }
        const bool live = (valid >> slot) & 1;
        float *weights = scratch + NQ * DP, *keeps = weights + kChunk * NQ;
        const int h0 = NQ == 1 ? 0 : half * kOwn;
#pragma unroll
        for (int g = 0; g < kOwn; g++) {
            const float v = live ? own[g] * unit : -INFINITY;
            if (z != nullptr && live && h0 + g < heads && (NQ > 1 || half == 0))
                z[int64_t(h0 + g) * stride + slot] = v;
            float top = v;
#pragma unroll
            for (int x = 8; x > 0; x >>= 1)
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
            const float next = fmaxf(m[g], top);
            const float keep = m[g] == next ? 1.0f : exp2f(m[g] - next);
            m[g] = next;
            const float w = exp2f(v - (next == -INFINITY ? 0.0f : next));
            l[g] = l[g] * keep + w;
            weights[slot * NQ + h0 + g] = w;
            if (slot == 0)
                keeps[h0 + g] = keep;
        }
        __syncwarp();
        const int piece = lane % kLanes, share = lane / kLanes;
        float keep[NQ];
#pragma unroll
        for (int g = 0; g < NQ; g++)
            keep[g] = keeps[g];
#pragma unroll
        for (int g = 0; g < NQ; g++)
#pragma unroll
            for (int n = 0; n < kPieces; n++)
#pragma unroll
                for (int j = 0; j < 4; j++)
                    o[g][n][j] *= keep[g];
#pragma unroll 4
        for (int t = share; t < kChunk; t += kShares) {
            float w[NQ];
#pragma unroll
            for (int g = 0; g < NQ; g++)
                w[g] = weights[t * NQ + g];
#pragma unroll
            for (int n = 0; n < kPieces; n++) {
                if (piece + n * kLanes >= kQuads)
                    break;
                const int c = piece + n * kLanes;
                const float4 v = *reinterpret_cast<const float4 *>(stage + (kBlocks + (c >> 3)) * kBlock + t * 128 +
                                                                   (((c & 7) ^ (t & 7)) << 4));
#pragma unroll
                for (int g = 0; g < NQ; g++) {
                    o[g][n][0] = fmaf(w[g], v.x, o[g][n][0]);
                    o[g][n][1] = fmaf(w[g], v.y, o[g][n][1]);
                    o[g][n][2] = fmaf(w[g], v.z, o[g][n][2]);
                    o[g][n][3] = fmaf(w[g], v.w, o[g][n][3]);
                }
            }
        }
        __syncwarp(); /* weights are overwritten by the next step */
    }

    __device__ __forceinline__ void statistics(float *maxima, float *sums) {
        const int lane = threadIdx.x & 31, half = lane >> 4;
#pragma unroll
        for (int g = 0; g < kOwn; g++) {
#pragma unroll
            for (int x = 8; x > 0; x >>= 1)
                l[g] += __shfl_xor_sync(0xffffffffu, l[g], x);
            const int h = (NQ == 1 ? 0 : half * kOwn) + g;
            if ((lane & 15) == 0 && (NQ > 1 || half == 0)) {
                maxima[h] = m[g];
                sums[h] = l[g];
            }
        }
    }
    template <bool kAdd> __device__ __forceinline__ void output(float *out, const float *factor) {
        const int lane = threadIdx.x & 31, piece = lane % kLanes, share = lane / kLanes;
#pragma unroll
        for (int g = 0; g < NQ; g++) {
            const float f = factor[g];
#pragma unroll
            for (int n = 0; n < kPieces; n++) {
#pragma unroll
                for (int j = 0; j < 4; j++)
#pragma unroll
                    for (int x = kLanes; x < 32; x <<= 1)
                        o[g][n][j] += __shfl_xor_sync(0xffffffffu, o[g][n][j], x);
                if (share == 0 && piece + n * kLanes < kQuads) {
                    float4 *to = reinterpret_cast<float4 *>(out + g * DP + (piece + n * kLanes) * 4);
                    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    if (f != 0.0f)
                        v = make_float4(o[g][n][0] * f, o[g][n][1] * f, o[g][n][2] * f, o[g][n][3] * f);
                    if (kAdd) {
                        const float4 u = *to;
                        v = make_float4(v.x + u.x, v.y + u.y, v.z + u.z, v.w + u.w);
                    }
                    *to = v;
                }
            }
        }
    }
};

template <typename Op> struct Scratch {
    static constexpr int value = 0;
};
template <int NQ, int DP> struct Scratch<Wide<NQ, DP>> {
    static constexpr int value = (Wide<NQ, DP>::kScratch + 3) / 4 * 4;
};

/* Stages of a warp's ring.  With 8 KB stages, three and two CTAs an SM stream
 * from HBM faster than two and three CTAs (100 against 103 us for 545 MB, 57
 * against 59.5 for 250 MB of listed pages); out of L2 it is the other way round
 * (129 against 115.5 us for 2.1 GB). */
constexpr int stages_of(int stage_bytes) { return stage_bytes <= 4096 ? 4 : stage_bytes <= 12288 ? 3 : 2; }

/* Shared memory: each warp's ring of stages and scratch, and two outputs of
 * [8][DP] in which the warps' states meet. */
template <typename Op> struct Plan {
    static constexpr int kStages = stages_of(Op::kStageBytes);
    static constexpr int kRing = kStages * Op::kStageBytes;
    static constexpr int kScratchBytes = Scratch<Op>::value * 4;
    static constexpr int kWarps = Op::kWarps, kThreads = kWarps * 32;
    static constexpr int kTile = kWarps * kChunk; /* slots of a tile */
    static constexpr int kOutputBytes = kRows * Op::DP * 4;
    static constexpr int kBytes = kWarps * (kRing + kScratchBytes) + 2 * kOutputBytes + 1024; /* to align */
    static constexpr int kFit = 228 * 1024 / (kBytes + 2048);
    static constexpr int kPerSm = kFit < Op::kMaxPerSm ? (kFit > 1 ? kFit : 1) : Op::kMaxPerSm;
    static_assert(kWarps * kRing >= kMaxSms * kPerSm * kRows * 4 + 128 + kOutputBytes + 2 * kRows * 4,
                  "the factors of an item's parts and one part fit there");
};

/* Slots of a row that the kernel walks: its length, or the listed pages. */
__device__ __forceinline__ int walked(const PagedAttention &a, int length) {
    return length == 0 ? 0 : a.selected ? a.n_selected * a.p.page_size : length;
}

template <typename R> __device__ __forceinline__ void store4(R *to, float4 v) {
    to[0] = output_of<R>(v.x);
    to[1] = output_of<R>(v.y);
    to[2] = output_of<R>(v.z);
    to[3] = output_of<R>(v.w);
}

/* Joins the `parts` parts of an item left by CTAs c0, c0 + 1, ...; run by
 * the whole CTA that arrived last.  Bulk copies bring the parts to shared
 * memory, and the warps turn their maxima and sums into one factor
 * exp(m_c - m) / l per part and head.  (Read by one load after another, 37
 * parts cost 200 us; with sixteen in flight a thread, 7.)  */
template <typename R, int DP, int kWarps>
__device__ __noinline__ void join_parts(const PagedAttention &a, bool inside, int c0, int parts, int r,
                                        int first_head, int heads, char *space, int bytes, uint64_t *bar,
                                        uint32_t &phase) {
    constexpr int kPartialFloats = paged_part_floats(DP);
    const PagedPool &p = a.p;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    /* an item that starts inside its first CTA's share lies in that one's second slot */
    const float *first = a.partial + (int64_t(c0) * 2 + (inside ? 1 : 0)) * kPartialFloats;
    const float *rest = a.partial + (int64_t(c0) * 2 + 2) * kPartialFloats;
    auto part = [&](int c) { return c == 0 ? first : rest + int64_t(c - 1) * 2 * kPartialFloats; };
    float *factor = reinterpret_cast<float *>(space);
    const int head_room = (parts * kRows * 4 + 127) / 128 * 128;
    const int size = (2 * kRows + heads * DP) * 4, pitch = size / 4; /* of a part */
    const int most = (bytes - head_room) / size;
    float *copies = reinterpret_cast<float *>(space + head_room);
    auto fetch = [&](int c, int n) { /* by warp 0 */
        fence_proxy_async(); /* others' stores, seen by this thread, before its copies */
        if (lane == 0)
            mbar_expect_tx(bar, n * size);
        __syncwarp();
        for (int k = lane; k < n; k += 32)
            bulk_g2s(copies + k * pitch, part(c + k), size, bar);
    };
    if (warp == 0)
        fetch(0, min(parts, most));
    const bool fit = parts <= most; /* then the statistics are read from the copies too */
    if (!stage_wait(bar, phase)) {
        paged_fail(p, kPagedTimeout);
        stage_wait(bar, phase); /* once more before its place is used again */
    }
    phase ^= 1;
    auto statistic = [&](int c, int i) { return fit ? copies[c * pitch + i] : __ldcg(part(c) + i); };
    for (int g = warp; g < heads; g += kWarps) {
        float top = -INFINITY, sum = 0.0f;
        for (int c = lane; c < parts; c += 32)
            top = fmaxf(top, statistic(c, g));
        top = warp_max(top);
        const float base = top == -INFINITY ? 0.0f : top;
        for (int c = lane; c < parts; c += 32) {
            const float f = exp2f(statistic(c, g) - base), l = statistic(c, kRows + g);
            factor[c * kRows + g] = f;
            sum = l != 0.0f ? fmaf(l, f, sum) : sum;
        }
        sum = warp_sum(sum);
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        for (int c = lane; c < parts; c += 32)
            factor[c * kRows + g] *= inv;
        if (lane == 0) {
            const float lse2 = sum == 0.0f ? -INFINITY : top + log2f(sum);
            if (a.lse)
                a.lse[int64_t(r) * p.heads + first_head + g] = lse2 * kLn2;
            if (a.weights)
                a.lse2[int64_t(r) * p.heads + first_head + g] = lse2;
        }
    }
    __syncthreads();
    constexpr int kQuads = (kRows * DP / 4 + kWarps * 32 - 1) / (kWarps * 32); /* 4-dim pieces a thread may have */
    float4 o[kQuads];
#pragma unroll
    for (int q = 0; q < kQuads; q++)
        o[q] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int c = 0; c < parts; c += most) {
        const int n = min(parts - c, most);
        if (c > 0) {
            if (!stage_wait(bar, phase)) {
                paged_fail(p, kPagedTimeout);
                stage_wait(bar, phase);
            }
            phase ^= 1;
        }
#pragma unroll
        for (int q = 0; q < kQuads; q++) {
            const int i = (q * kWarps * 32 + tid) * 4, g = i / DP;
            if (g < heads)
                for (int k = 0; k < n; k++) {
                    const float4 x = *reinterpret_cast<const float4 *>(copies + k * pitch + 2 * kRows + i);
                    const float f = factor[(c + k) * kRows + g];
                    o[q].x = fmaf(x.x, f, o[q].x);
                    o[q].y = fmaf(x.y, f, o[q].y);
                    o[q].z = fmaf(x.z, f, o[q].z);
                    o[q].w = fmaf(x.w, f, o[q].w);
                }
        }
        __syncthreads();
        if (warp == 0 && c + n < parts)
            fetch(c + n, min(parts - c - n, most));
    }
#pragma unroll
    for (int q = 0; q < kQuads; q++) {
        const int i = (q * kWarps * 32 + tid) * 4, g = i / DP, d = i % DP;
        if (g < heads && d < p.head_dim)
            store4<R>(static_cast<R *>(a.out) + r * a.out_stride + int64_t(first_head + g) * p.head_dim + d, o[q]);
    }
}

/* An item of so many tiles takes up this much of the line: its tiles come
 * behind kItemCost places without one. */
__device__ __forceinline__ int line_of(int tiles) { return tiles == 0 ? 0 : tiles + kItemCost; }

/* One item, or the part of it that lies in a CTA's share. */
struct Item {
    int row, sequence, length, span, tiles, index; /* index within the row */
    int tile, tile0, tile1;
    int first; /* where its first tile lies on the line */
};

/* Walks the items of a share. */
struct Cursor {
    int pos, last, in_row; /* place on the line, end, place within the row's items */
    int r;

    __device__ __forceinline__ bool next(const PagedAttention &a, int items_per_row, int tile_slots, Item &x) {
        while (pos < last) {
            x.sequence = row_span(a.p, a.row_sequence, a.row_length, r, x.length);
            x.span = walked(a, x.length);
            x.tiles = (x.span + tile_slots - 1) / tile_slots;
            if (x.tiles == 0) {
                r++;
                continue;
            }
            const int len = line_of(x.tiles);
            x.index = in_row / len;
            const int place = in_row - x.index * len;
            const int taken = min(len - place, last - pos);
            x.row = r;
            x.tile = x.tile0 = max(place - kItemCost, 0);
            x.tile1 = place + taken - kItemCost;
            x.first = pos - place + kItemCost;
            pos += taken;
            in_row += taken;
            if (in_row >= len * items_per_row) {
                in_row = 0;
                r++;
            }
            if (x.tile1 > x.tile0)
                return true;
        }
        return false;
    }
};

/* Logits of a box of slots whose page is a bad one: they give no weight.  By
 * the lane that found it; where the logits are made it would cost the kernel
 * registers (42 against 39 us for 16 sequences of up to 4,096 slots, bf16,
 * fp32 rows). */
__device__ __noinline__ void no_weight(const PagedAttention &a, int row, int index, int slot) {
    const PagedPool &p = a.p;
    const int groups = (p.group + kRows - 1) / kRows, in_group = index % groups * kRows;
    float *z = a.logits + (int64_t(row) * p.heads + index / groups * p.group + in_group) * p.capacity + slot;
    for (int g = 0; g < min(kRows, p.group - in_group); g++)
        for (int i = 0; i < a.box; i++)
            z[int64_t(g) * p.capacity + i] = -INFINITY;
}

/* Places of one of row r's items. */
__device__ __noinline__ int places_of(const PagedAttention &a, int r, int tile_slots) {
    int length;
    row_span(a.p, a.row_sequence, a.row_length, r, length);
    return line_of((walked(a, length) + tile_slots - 1) / tile_slots);
}

/* kLean: pages of whole 16-slot chunks, rows of whole columns, no weights
 * asked for.  Without the run-time forms of these the loop is shorter (sparse
 * prompt 130 against 140 us, sparse short 12.7 against 13.4). */
template <typename Op, typename R, bool kLean>
__global__ void __launch_bounds__(Plan<Op>::kThreads, Plan<Op>::kPerSm)
    attention_kernel(const __grid_constant__ PagedAttention a) {
    using T = typename Op::Cache;
    constexpr int DP = Op::DP, kStages = Plan<Op>::kStages, kWarps = Plan<Op>::kWarps,
                  kThreads = Plan<Op>::kThreads, kTile = Plan<Op>::kTile;
    extern __shared__ char smem_raw[];
    char *smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    __shared__ uint32_t masks[kWarps][kStages];
    __shared__ uint64_t full[kWarps][kStages], joined;
    __shared__ float maxima[2][kWarps][kRows], sums[2][kWarps][kRows], factors[kWarps][kRows];
    __shared__ int warp_sums[kWarps], found_row, found_place, arrived_last[2];
    __shared__ Item shared[2]; /* items that other CTAs have parts of: the first and the last at most */
    const PagedPool &p = a.p;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int groups = (p.group + kRows - 1) / kRows, items_per_row = p.kv_heads * groups;

    if (tid == 0) {
        for (int i = 0; i < kWarps * kStages; i++)
            mbar_init(&full[0][0] + i, 1);
        mbar_init(&joined, 1);
        fence_barrier_init();
    }
    begin_kernel();

    /* this CTA's share of the line of tiles: thread i sums a run of rows */
    const int run = (a.rows + kThreads - 1) / kThreads;
    const int r0 = min(tid * run, a.rows), r1 = min(r0 + run, a.rows);
    int mine = 0;
#pragma unroll 1
    for (int r = r0; r < r1; r++)
        mine += places_of(a, r, kTile);
    int upto = mine;
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, upto, x);
        upto += lane >= x ? v : 0;
    }
    if (lane == 31)
        warp_sums[warp] = upto;
    __syncthreads();
    int total = 0;
#pragma unroll
    for (int w = 0; w < kWarps; w++) {
        upto += w < warp ? warp_sums[w] : 0;
        total += warp_sums[w];
    }
    total *= items_per_row;
    const int share = (total + int(gridDim.x) - 1) / int(gridDim.x), start = int(blockIdx.x) * share;
    int at = (upto - mine) * items_per_row;
    if (start < total && start >= at && start < upto * items_per_row)
#pragma unroll 1
        for (int r = r0; r < r1; r++) {
            const int n = run == 1 ? mine * items_per_row : places_of(a, r, kTile) * items_per_row;
            if (start < at + n) {
                found_row = r;
                found_place = start - at;
                break;
            }
            at += n;
        }
    __syncthreads();

    char *ring = smem + warp * Plan<Op>::kRing;
    const uint32_t ring_at = smem_u32(ring);
    float *scratch = reinterpret_cast<float *>(smem + kWarps * Plan<Op>::kRing + warp * Plan<Op>::kScratchBytes);
    float *outputs = reinterpret_cast<float *>(smem + kWarps * (Plan<Op>::kRing + Plan<Op>::kScratchBytes));
    const int D = p.head_dim, box = kLean ? kChunk : a.box, boxes = kLean ? 1 : kChunk / box;
    constexpr int kBoxWidth = 128 / sizeof(T);
    uint32_t phases = 0;
    uint32_t late = 0; /* stages whose copy did not arrive: then nothing more is read */

    /* The copies run ahead of the arithmetic by kStages - 1 chunks, through
     * the ends of items: under load a round trip to memory takes 3 us, and an
     * item that began with empty stages cost 10 to 20. */
    Cursor feed{start, min(start + share, total), found_place, found_row}, eat = feed;
    Item in, x;
    bool more = feed.next(a, items_per_row, kTile, in);

    /* Where this warp's chunks of the next 32 / boxes tiles of an item lie, a
     * box a lane (box i of chunk k in lane k boxes + i), and how many of a
     * box's slots count.  One look-up, two round trips long, serves that many
     * chunks, and is made that many ahead. */
    struct Batch {
        int page, slot, count, tiles, head;
    };
    const int my_chunk = lane / boxes, my_box = lane - my_chunk * boxes;
    auto plan = [&](Batch &b) {
        b.count = b.tiles = 0;
        if (!more)
            return;
        const int v = (in.tile + my_chunk) * kTile + warp * kChunk + my_box * box;
        b.tiles = min(32 / boxes, in.tile1 - in.tile);
        b.head = in.index / groups;
        if (my_chunk < b.tiles && v < in.span) {
            int j = int((uint64_t(unsigned(v)) * a.page_magic) >> a.page_shift);
            b.slot = v - j * p.page_size;
            bool there = true;
            if (a.selected) {
                j = a.selected[(int64_t(in.row) * p.kv_heads + b.head) * a.n_selected + j];
                there = j >= 0 && j < p.max_pages && j * p.page_size + b.slot < in.length;
            }
            if (there) {
                b.page = checked_page(p, in.sequence, j);
                if (b.page >= 0)
                    b.count = min(box, in.length - j * p.page_size - b.slot);
                else if (!kLean && a.weights)
                    no_weight(a, in.row, in.index, v);
            }
        }
        in.tile += b.tiles;
        if (in.tile == in.tile1) {
            more = feed.next(a, items_per_row, kTile, in);
            if (more && warp == 0) { /* its queries, on their way to L2 */
                const char *q = reinterpret_cast<const char *>(
                    static_cast<const R *>(a.q) + in.row * a.q_stride +
                    int64_t(in.index / groups * p.group + in.index % groups * kRows) * D);
                if (lane * 128 < min(kRows, p.group - in.index % groups * kRows) * D * int(sizeof(R)))
                    asm volatile("prefetch.global.L2 [%0];\n" ::"l"(q + lane * 128));
            }
        }
    };
    Batch now{}, then{};
    int used = 0; /* chunks of `now` that have been issued */
    auto issue = [&](int stage) {
        if (used == now.tiles) {
            now = then;
            used = 0;
            plan(then);
        }
        const uint32_t to = ring_at + stage * Op::kStageBytes + my_box * box * 128;
        const bool mine = now.count > 0 && my_chunk == used && late == 0;
        const uint32_t valid = __reduce_or_sync(0xffffffffu, mine ? ((1u << now.count) - 1u) << (my_box * box) : 0u);
        const uint32_t bar = smem_u32(&full[warp][stage]);
        if (boxes > 1) {
            const int n = __popc(__ballot_sync(0xffffffffu, mine));
            if (lane == 0) {
                masks[warp][stage] = valid;
                if (n > 0)
                    mbar_expect_tx(&full[warp][stage], n * box * 128 * 2 * Op::kBlocks);
            }
            __syncwarp();
        } else {
            if (lane == 0)
                masks[warp][stage] = valid;
            if (mine)
                mbar_expect_tx(&full[warp][stage], Op::kStageBytes);
        }
        if (mine) {
            if (kLean || a.whole_columns) {
                copy_box(to, &a.key_map, 0, now.slot, 0, now.head, now.page, bar);
                copy_box(to + Op::kBlocks * kBlock, &a.value_map, 0, now.slot, 0, now.head, now.page, bar);
            } else {
#pragma unroll
                for (int b = 0; b < Op::kBlocks; b++) {
                    copy_box(to + b * kBlock, &a.key_map, b * kBoxWidth, now.slot, 0, now.head, now.page, bar);
                    copy_box(to + (Op::kBlocks + b) * kBlock, &a.value_map, b * kBoxWidth, now.slot, 0, now.head,
                             now.page, bar);
                }
            }
        }
        if (used < now.tiles)
            used++;
    };

    plan(now);
    plan(then);
    for (int i = 0; i < kStages - 1; i++)
        issue(i);
    __syncwarp(); /* lane 0's masks, for all lanes */

    /* rows that see nothing */
    for (int r = blockIdx.x; r < a.rows; r += gridDim.x) {
        int length;
        row_span(p, a.row_sequence, a.row_length, r, length);
        if (length != 0)
            continue;
        for (int i = tid; i < p.heads * p.head_dim; i += kThreads)
            static_cast<R *>(a.out)[r * a.out_stride + i] = from_float<R>(0.0f);
        for (int h = tid; h < p.heads; h += kThreads)
            if (a.lse)
                a.lse[int64_t(r) * p.heads + h] = -INFINITY;
    }

    int stage = 0, turn = 0, parts = 0;
    while (eat.next(a, items_per_row, kTile, x)) {
        const int first_head = x.index / groups * p.group + x.index % groups * kRows;
        const int heads = min(kRows, p.group - x.index % groups * kRows);
        Op op;
        op.begin(a, static_cast<const R *>(a.q) + x.row * a.q_stride + int64_t(first_head) * D, heads, scratch);
        for (; x.tile < x.tile1; x.tile++) {
            issue(stage == 0 ? kStages - 1 : stage - 1);
            const uint32_t valid = masks[warp][stage];
            bool arrived = valid != 0;
            if (arrived) {
                /* the lanes give up together: what follows needs the whole warp */
                arrived = __all_sync(0xffffffffu, stage_wait(&full[warp][stage], (phases >> stage) & 1));
                if (arrived) {
                    phases ^= 1u << stage;
                } else {
                    paged_fail(p, kPagedTimeout);
                    late |= 1u << stage;
                }
            }
            if (arrived) {
                const uint32_t at = ring_at + stage * Op::kStageBytes;
                if (valid != 0xffffu) {
                    /* values that do not count meet weights of 0: they must be finite */
                    for (int i = lane; i < kChunk * 8 * Op::kBlocks; i += 32)
                        if (!((valid >> (i / 8 % kChunk)) & 1))
                            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};\n" ::"r"(
                                             at + Op::kBlocks * kBlock + i * 16),
                                         "r"(0)
                                         : "memory");
                    __syncwarp();
                }
                float *z = !kLean && a.weights ? a.logits + (int64_t(x.row) * p.heads + first_head) * p.capacity +
                                           x.tile * kTile + warp * kChunk
                                     : nullptr;
                op.step(at, valid, scratch, z, p.capacity, heads);
                if (valid != 0xffffu)
                    fence_async(); /* the zeros, before the stage is filled again */
            }
            __syncwarp();
            stage = stage + 1 == kStages ? 0 : stage + 1;
        }

        /* the warps' states meet: a common maximum, then outputs in a fixed
         * order, two warps at a time */
        float(&top)[kWarps][kRows] = maxima[turn], (&sum)[kWarps][kRows] = sums[turn];
        turn ^= 1;
        op.statistics(top[warp], sum[warp]);
        __syncthreads();
        float(&factor)[kRows] = factors[warp];
        const bool whole = x.tile0 == 0 && x.tile1 == x.tiles;
        float *part = a.partial + (int64_t(blockIdx.x) * 2 + (x.first <= start ? 0 : 1)) * paged_part_floats(DP);
        if (lane < kRows) {
            float m = -INFINITY, l = 0.0f;
#pragma unroll
            for (int w = 0; w < kWarps; w++)
                m = fmaxf(m, top[w][lane]);
            const float base = m == -INFINITY ? 0.0f : m;
#pragma unroll
            for (int w = 0; w < kWarps; w++)
                l = fmaf(sum[w][lane], exp2f(top[w][lane] - base), l);
            /* a whole item's outputs are divided by the sum here */
            const float inv = !whole ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
            factor[lane] = exp2f(top[warp][lane] - base) * inv;
            if (warp == 0 && lane < heads) {
                if (whole) {
                    const float lse2 = l == 0.0f ? -INFINITY : m + log2f(l);
                    const int64_t at = int64_t(x.row) * p.heads + first_head + lane;
                    if (a.lse)
                        a.lse[at] = lse2 * kLn2;
                    if (a.weights)
                        a.lse2[at] = lse2;
                } else {
                    part[lane] = m;
                    part[kRows + lane] = l;
                }
            }
        }
        __syncwarp();
        if (warp < 2)
            op.template output<false>(outputs + warp * kRows * DP, factor);
        __syncthreads();
#pragma unroll
        for (int w = 2; w < kWarps; w += 2) {
            if (warp / 2 == w / 2)
                op.template output<true>(outputs + warp % 2 * kRows * DP, factor);
            __syncthreads();
        }
        for (int i = tid; i < heads * (DP / 4); i += kThreads) {
            const int g = i / (DP / 4), d = i % (DP / 4) * 4;
            const float4 u = *reinterpret_cast<const float4 *>(outputs + g * DP + d);
            const float4 v = *reinterpret_cast<const float4 *>(outputs + (kRows + g) * DP + d);
            const float4 o = make_float4(u.x + v.x, u.y + v.y, u.z + v.z, u.w + v.w);
            if (!whole)
                *reinterpret_cast<float4 *>(part + 2 * kRows + g * DP + d) = o;
            else if (d < D)
                store4<R>(static_cast<R *>(a.out) + x.row * a.out_stride + int64_t(first_head + g) * D + d, o);
        }
        if (!whole) {
            if (tid == 0)
                shared[parts] = x;
            parts++;
        }
        __syncthreads(); /* outputs and factors are free again */
    }
    for (; late != 0; late &= late - 1) /* once more, before the stages are used again */
        stage_wait(&full[warp][__ffs(late) - 1], (phases >> (__ffs(late) - 1)) & 1);
    if (parts == 0)
        return;

    /* of items shared with other CTAs, the last to arrive joins the parts */
    __syncthreads();
    if (tid < parts) {
        const Item &y = shared[tid];
        int *counter = a.counters + int64_t(y.row) * items_per_row + y.index, before_me;
        const int others = (y.first + y.tiles - 1) / share - y.first / share;
        /* releases the block's parts (ordered before by the barrier) and
         * acquires the others' */
        asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;\n" : "=r"(before_me) : "l"(counter) : "memory");
        arrived_last[tid] = before_me == others;
        if (before_me == others)
            *counter = 0;
    }
    __syncthreads();
    uint32_t join_phase = 0;
    for (int i = 0; i < parts; i++)
        if (arrived_last[i]) {
            const Item &y = shared[i];
            const int c0 = y.first / share, c1 = (y.first + y.tiles - 1) / share;
            join_parts<R, DP, kWarps>(a, y.first > c0 * share, c0, c1 - c0 + 1, y.row,
                                      y.index / groups * p.group + y.index % groups * kRows,
                                      min(kRows, p.group - y.index % groups * kRows), smem, kWarps * Plan<Op>::kRing,
                                      &joined, join_phase);
            __syncthreads();
        }
}

/* weights_out[t] = weights[t] + sum over the group of exp(z_t - lse): every
 * slot has one writer, so the order of the sum is fixed.  Four slots a
 * thread; kVec: their addresses are multiples of 16 bytes. */
constexpr int kWeightThreads = 256;

template <bool kVec>
__global__ void __launch_bounds__(kWeightThreads) weights_kernel(const __grid_constant__ PagedAttention a) {
    begin_kernel();
    const PagedPool &p = a.p;
    const int head = blockIdx.y, r = blockIdx.z;
    int length;
    row_span(p, a.row_sequence, a.row_length, r, length);
    const int t = (int(blockIdx.x) * kWeightThreads + int(threadIdx.x)) * 4;
    if (t >= length)
        return;
    const int error = *p.error;
    const int64_t to = (int64_t(r) * p.kv_heads + head) * p.capacity + t;
    const int64_t h0 = int64_t(r) * p.heads + head * p.group;
    const float *z = a.logits + h0 * p.capacity + t;
    const int n = min(4, length - t);
    float w[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int g = 0; g < p.group; g++) {
        float lse2 = a.lse2[h0 + g];
        if (lse2 == -INFINITY) /* every logit was: the head sees nothing */
            lse2 = INFINITY;
        float x[4];
        if constexpr (kVec) {
            *reinterpret_cast<float4 *>(x) = *reinterpret_cast<const float4 *>(z + int64_t(g) * p.capacity);
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++)
                x[i] = i < n ? z[int64_t(g) * p.capacity + i] : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < 4; i++)
            w[i] += exp2f(x[i] - lse2);
    }
    if (error & kPagedTimeout) /* logits may be missing */
        return;
    if (kVec && n == 4) {
        const float4 x = *reinterpret_cast<const float4 *>(a.weights + to);
        *reinterpret_cast<float4 *>(a.weights_out + to) =
            make_float4(x.x + w[0], x.y + w[1], x.z + w[2], x.w + w[3]);
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (i < n)
            a.weights_out[to + i] = a.weights[to + i] + w[i];
}

template <typename Op, typename R>
cudaError_t launch(const PagedAttention &a, cudaStream_t s) {
    constexpr int bytes = Plan<Op>::kBytes, threads = Plan<Op>::kThreads, tile = Plan<Op>::kTile;
    static_assert(bytes <= 227 * 1024, "stages exceed the SM's shared memory");
    constexpr bool kHasLean = Op::DP != 96; /* 96 has no whole columns */
    const bool lean = kHasLean && a.box == kChunk && a.whole_columns && !a.weights;
    const auto kernel = lean ? attention_kernel<Op, R, kHasLean> : attention_kernel<Op, R, false>;
    static int fit[2][kMaxDevices] = {};
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess)
        return e;
    int &per_sm = fit[lean][device % kMaxDevices];
    if (per_sm == 0) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (e != cudaSuccess)
            return e;
        int n = 0;
        e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, threads, bytes);
        if (e != cudaSuccess)
            return e;
        per_sm = n < 1 ? 1 : n > Plan<Op>::kPerSm ? Plan<Op>::kPerSm : n;
    }
    const PagedPool &p = a.p;
    const int64_t items = int64_t(a.rows) * p.kv_heads * ((p.group + kRows - 1) / kRows);
    const int64_t slots = a.selected ? int64_t(a.n_selected) * p.page_size : p.capacity;
    const int64_t tiles = items * ((slots + tile - 1) / tile);
    const int64_t ctas = int64_t(a.sms) * per_sm;
    e = launch_kernel(kernel, dim3(unsigned(tiles < ctas ? tiles : ctas)), threads, bytes, s, 1, a);
    if (e != cudaSuccess || !a.weights)
        return e;
    const unsigned blocks = unsigned((p.capacity + 4 * kWeightThreads - 1) / (4 * kWeightThreads));
    const uintptr_t bits = reinterpret_cast<uintptr_t>(a.weights) | reinterpret_cast<uintptr_t>(a.weights_out) |
                           uintptr_t(p.capacity) * 4;
    return launch_kernel((bits & 15) == 0 ? weights_kernel<true> : weights_kernel<false>,
                         dim3(blocks, p.kv_heads, a.rows), kWeightThreads, 0, s, 1, a);
}

template <typename T, typename R> cudaError_t launch_halves(const PagedAttention &a, cudaStream_t s) {
    switch (paged_padded_dim(a.p.type, a.p.head_dim)) {
    case 64:
        return launch<Halves<T, R, 64>, R>(a, s);
    case 96:
        return launch<Halves<T, R, 96>, R>(a, s);
    case 128:
        return launch<Halves<T, R, 128>, R>(a, s);
    case 192:
        return launch<Halves<T, R, 192>, R>(a, s);
    default:
        return launch<Halves<T, R, 256>, R>(a, s);
    }
}

template <int NQ> cudaError_t launch_wide(const PagedAttention &a, cudaStream_t s) {
    switch (paged_padded_dim(a.p.type, a.p.head_dim)) {
    case 32:
        return launch<Wide<NQ, 32>, float>(a, s);
    case 64:
        return launch<Wide<NQ, 64>, float>(a, s);
    case 128:
        return launch<Wide<NQ, 128>, float>(a, s);
    default:
        return launch<Wide<NQ, 256>, float>(a, s);
    }
}

} // namespace

cudaError_t paged_attention(const PagedAttention &a, cudaStream_t s) {
    if (a.p.type == 0)
        return a.p.group == 1 ? launch_wide<1>(a, s) : a.p.group <= 4 ? launch_wide<4>(a, s) : launch_wide<8>(a, s);
    if (a.p.type == 1)
        return a.type == 0 ? launch_halves<__half, float>(a, s) : launch_halves<__half, __half>(a, s);
    return a.type == 0 ? launch_halves<__nv_bfloat16, float>(a, s)
                       : launch_halves<__nv_bfloat16, __nv_bfloat16>(a, s);
}

} // namespace nut
