/* Attention of drafted tokens over a 16-bit paged KV cache on the tensor cores
 * (nut_paged_tree_attention, head_dim up to 128).
 *
 * All rows of a sequence that share a kv head (drafted tokens by query heads)
 * are one matrix, so a pass over the cache serves them together: logits
 * S = Q K^T and outputs O += P V of 128 rows by tcgen05.mma, with S, P and O in
 * tensor memory and a thread for each row in the softmax between them.
 *
 *   warps 0-3   the softmax, a thread for each row
 *   warp 4      copies key and value tiles of 64 slots (TMA boxes of a page's
 *               slots) into a ring of stages, and notes which slots there are
 *   warp 5      issues the products: those of the next tile's logits run
 *               during the softmax
 * Two such blocks share an SM where the queries leave room: one's products
 * and copies run while the other is in its softmax, loads its queries or
 * writes its outputs.
 *
 * Queries in fp32 are split into 16-bit terms that multiply the same keys, and
 * so are their weights: two for fp16 (queries first scaled by a power of two
 * to [2^10, 2^11)), three for bf16.  Weights are kept in the 16-bit type's
 * range by a power of two: of fp16 the greatest is 2^8 to 2^15, since fp16 ends
 * at 2^-24; of bf16 it is 2^-30 at most, so that no sum of values near bf16's
 * greatest overflows.  A row's maximum may lag behind by kSlack: its outputs
 * are rescaled only when it rises by more.
 *
 * Sums in tensor memory are cut off, not rounded: over a thousand products a
 * row of outputs comes out short by 4 to 8 parts in 10^5, less than a 16-bit
 * output's rounding (200,000 slots in one block would reach fp16's half step),
 * but not an fp32 one's.  fp32 rows therefore take a tile's
 * product at a time, which the softmax of the next tile adds, rounded to
 * nearest, to what it has put aside (kAside), and small terms are multiplied
 * first.  With and without: 32 caches of up to 4,096 slots, 32/8 heads, 16
 * tokens, fp16 of 64 dims 77.5 and 79.7 us, of 128 dims 135 and 128.5, bf16 of
 * 64 dims 99 and 94.5, of 128 dims 163 and 160.5.
 *
 * Rows of the cache's type have weights in one term.  Two would bring the error
 * down to that of rounding the outputs (bf16: 2.2 in place of 3.0 x 10^-4, root
 * mean square), and take 85 us where the batch below takes 72 after a flush of
 * L2.  A caller who wants them passes fp32 rows.
 *
 * Values of slots that some rows do not see would meet weights of 0 in the
 * product: among the drafted tokens infinities and NaN are taken out of the
 * tile, and added at the end to the rows that see them.
 *
 * What bounds it: HBM and the latency of a share.  32 bf16 caches of up to
 * 4,096 slots (282 MB, 8 kv heads of 128 dims, 16 tokens each): 65 us, 4.4
 * TB/s of DRAM over all of it; within a share its tiles come at 5.7 to 6 TB/s,
 * 5 us go by before the first, 3 us on an item's way out, and 8 us to the
 * joining of parts (launched behind, partly beside).  One block an SM on tiles
 * of 128 slots took 144 us: its copies and products stood still in the
 * softmax.  Five stages of 16 KB in place of four gave nothing.  Two caches of
 * up to 60,000 slots with 33 tokens: 132 rows are two blocks of rows, each of
 * which reads the keys: 500 MB through the SMs in 100 us.
 */
#include <cstdint>
#include <type_traits>
#include <cuda_runtime.h>

#include "paged_tree.cuh"
#include "stream.cuh"

namespace nut {
namespace {

constexpr int kRows = 128;
constexpr int kTile = kTreeTile;
constexpr int kBuffers = 2; /* of logits */
constexpr int kProducer = 4, kIssuer = 5; /* warps */
constexpr int kThreads = 192;
constexpr uint64_t kTreeWaitNs = 2000000000ull;

/* kTerms: 16-bit terms of a query and of a weight. */
template <int DP_, int kTerms_> struct TcPlan {
    static constexpr int DP = DP_, kTerms = kTerms_;
    static constexpr int kColumns = DP / 64; /* of 128 bytes */
    static constexpr int kQueryBytes = kRows * DP * 2; /* of a term */
    static constexpr int kQueries = kQueryBytes * kTerms;
    static constexpr int kStage = kTile * DP * 2;
    static constexpr int kSpare = 1024 + 2560; /* alignment, static shared memory and the block's own 1 KB */
    static constexpr int kPerSm = kQueries + 4 * kStage + kSpare <= 114 * 1024 ? 2 : 1;
    static constexpr int kFit = ((kPerSm == 2 ? 114 : 227) * 1024 - kSpare - kQueries) / kStage;
    static constexpr int kStages = kFit < 12 ? kFit : 12;
    static constexpr int kBytes = 1024 + kQueries + kStages * kStage;
    /* tensor memory: S twice, two terms of P in its place; the third; O; what earlier tiles added to O.
     * Of that, dims that find no room are in registers */
    static constexpr int kMemory = kPerSm == 2 ? 256 : 512;
    static constexpr int kThird = 2 * kTile, kOutputs = kThird + (kTerms > 2 ? kTile / 2 : 0), kSums = kOutputs + DP;
    static constexpr bool kAside = kTerms > 1;
    static constexpr int kHeld = !kAside || kSums + DP <= kMemory ? 0 : kSums + DP - kMemory;
    static_assert(kSums + (kAside ? DP - kHeld : 0) <= kMemory && kHeld % 32 == 0 && kHeld < DP, "columns of tensor memory");
    static_assert(kQueries >= kRows * 128, "the outputs leave through there, 32 dims at a time");
    static_assert(kStages >= 4, "keys of two tiles and values of one are in use at a time");
    static_assert(kStages / 2 + 2 < 8, "tiles under way: Shared::valid");
    static_assert(kPerSm <= kTreeCtasPerSm, "the workspace has room for as many");
    template <typename T> static constexpr float lift() {
        return !std::is_same<T, __half>::value ? -38.0f : kTerms > 1 ? 15.0f : 8.0f;
    }
};

__host__ __device__ constexpr float power_of_two(int e) { return e == 0 ? 1.0f : e > 0 ? 2.0f * power_of_two(e - 1) : 0.5f * power_of_two(e + 1); }

/* ---- PTX --------------------------------------------------------------- */

__device__ __forceinline__ void copy_box(uint32_t to, const CUtensorMap *map, int x, int y, int b, int h, int w, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
                 "[%0], [%1, {%3, %4, %5, %6, %7}], [%2];\n" ::"r"(to),
                 "l"(map), "r"(bar), "r"(x), "r"(y), "r"(b), "r"(h), "r"(w)
                 : "memory");
}
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory"); }
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory"); }

/* D (+)= A B^T with both operands in shared memory, or A in tensor memory. */
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
                 "l"(a), "l"(b), "r"(idesc), "r"(uint32_t(add))
                 : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
                 "r"(a), "l"(b), "r"(idesc), "r"(uint32_t(add))
                 : "memory");
}

/* 32 columns of this warp's lanes of tensor memory; the loads are complete
 * after tc_wait_ld(). */
__device__ __forceinline__ void tmem_load32(uint32_t at, float *v) {
    uint32_t *r = reinterpret_cast<uint32_t *>(v);
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
                 "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
                 "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
                   "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
                   "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(at));
}
__device__ __forceinline__ void tmem_store16(uint32_t at, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
                 "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};\n" ::"r"(at),
                 "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
                 "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
                 : "memory");
}
__device__ __forceinline__ void tmem_store32(uint32_t at, const float *v) {
    const uint32_t *r = reinterpret_cast<const uint32_t *>(v);
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
                 "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
                 "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};\n" ::"r"(at),
                 "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
                 "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
                 "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
                 "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
                 : "memory");
}

/* 2^x, 0 below 2^-126. */
__device__ __forceinline__ float power2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}

/* A matrix in 128-byte rows with the 128-byte swizzle, 8 rows together.  Rows
 * along the product's M or N (K-major): 8 of them are `step` bytes from the
 * next 8, `lead` has no meaning.  Rows along its K (MN-major): 8 of K are
 * `step` bytes, 64 of N `lead`. */
__device__ __forceinline__ uint64_t matrix_at(uint32_t addr, uint32_t lead, uint32_t step) {
    return uint64_t((addr >> 4) & 0x3fffu) | uint64_t(lead >> 4) << 16 | uint64_t(step >> 4) << 32 | uint64_t(1) << 46 |
           uint64_t(2) << 61;
}
/* fp32 accumulators; fp16 or bf16 operands of 128 x K and N x K, B's rows along
 * K if `along_k`. */
template <typename T> __host__ __device__ constexpr uint32_t shape_of(int N, bool along_k) {
    return 1u << 4 | (std::is_same<T, __nv_bfloat16>::value ? 1u << 7 | 1u << 10 : 0u) | (along_k ? 1u << 16 : 0u) |
           uint32_t(N >> 3) << 17 | uint32_t(128 >> 4) << 24;
}

template <typename T> struct Pair;
template <> struct Pair<__half> {
    static constexpr uint32_t kInfinite = 0x7c00u;
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
    static __device__ __forceinline__ float2 unpack(uint32_t v) { return __half22float2(*reinterpret_cast<const __half2 *>(&v)); }
    static __device__ __forceinline__ uint32_t add_zero_times(uint32_t sum, uint32_t v) {
        asm("fma.rn.f16x2 %0, %1, %2, %0;\n" : "+r"(sum) : "r"(v), "r"(0u));
        return sum;
    }
};
template <> struct Pair<__nv_bfloat16> {
    static constexpr uint32_t kInfinite = 0x7f80u;
    static __device__ __forceinline__ uint32_t pack(float a, float b) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
    static __device__ __forceinline__ float2 unpack(uint32_t v) {
        return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
    }
    static __device__ __forceinline__ uint32_t add_zero_times(uint32_t sum, uint32_t v) {
        asm("fma.rn.bf16x2 %0, %1, %2, %0;\n" : "+r"(sum) : "r"(v), "r"(0u));
        return sum;
    }
};

/* ---- the kernel ---------------------------------------------------------- */

/* 16 bytes of elements whose address is a multiple of an element only.  (Not
 * through an array that a pointer reaches: that would lie in local memory, and
 * each of a thread's loads would wait for the one before.) */
__device__ __forceinline__ uint4 load_elements(const float *q) {
    return make_uint4(__float_as_uint(q[0]), __float_as_uint(q[1]), __float_as_uint(q[2]), __float_as_uint(q[3]));
}
template <typename R> __device__ __forceinline__ uint4 load_elements(const R *x) {
    const unsigned short *q = reinterpret_cast<const unsigned short *>(x);
    return make_uint4(q[0] | uint32_t(q[1]) << 16, q[2] | uint32_t(q[3]) << 16, q[4] | uint32_t(q[5]) << 16,
                      q[6] | uint32_t(q[7]) << 16);
}

/* Four outputs whose address is a multiple of an element only. */
template <typename R> __device__ __noinline__ void store_elements(R *to, float4 v, bool really) {
    if (really) {
        to[0] = output_of<R>(v.x);
        to[1] = output_of<R>(v.y);
        to[2] = output_of<R>(v.z);
        to[3] = output_of<R>(v.w);
    }
}
template <typename R> __device__ __forceinline__ uint32_t pack_outputs(float a, float b) {
    const R e[2] = {output_of<R>(a), output_of<R>(b)};
    return *reinterpret_cast<const uint32_t *>(e);
}

/* Takes infinities and NaN out of 16 bytes of values. */
template <typename T> __device__ __noinline__ void take_out(uint32_t at) {
    constexpr uint32_t kInf = Pair<T>::kInfinite;
    uint32_t e[4];
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];\n" : "=r"(e[0]), "=r"(e[1]), "=r"(e[2]), "=r"(e[3]) : "r"(at));
    for (int j = 0; j < 4; j++)
        e[j] &= ~__vcmpeq2(e[j] & (kInf | kInf << 16), kInf | kInf << 16);
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};\n" ::"r"(at), "r"(e[0]), "r"(e[1]), "r"(e[2]), "r"(e[3]) : "memory");
}

/* Half of a slot's row of a value tile, its 128-byte columns `lead` apart:
 * zeros where there is no such slot, else infinities and NaN taken out (and
 * noted).  0 times a value is NaN if it is one of those. */
template <typename T, int DP>
__device__ __forceinline__ void clean_values(uint32_t row, int slot, int half, uint32_t lead, bool there, int *odd) {
    constexpr int kPieces = DP / 16;
    const auto at = [&](int k) {
        const int c = half * kPieces + k;
        return row + (c >> 3) * lead + (((c & 7) ^ (slot & 7)) << 4);
    };
    if (!there) {
#pragma unroll
        for (int k = 0; k < kPieces; k++)
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};\n" ::"r"(at(k)), "r"(0) : "memory");
        return;
    }
    uint32_t zeros[4] = {0, 0, 0, 0};
#pragma unroll
    for (int k = 0; k < kPieces; k++) {
        uint32_t e[4];
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];\n" : "=r"(e[0]), "=r"(e[1]), "=r"(e[2]), "=r"(e[3]) : "r"(at(k)));
#pragma unroll
        for (int j = 0; j < 4; j++)
            zeros[j] = Pair<T>::add_zero_times(zeros[j], e[j]);
    }
    const uint32_t all = (zeros[0] | zeros[1] | zeros[2] | zeros[3]) & 0x7fff7fffu;
    if (all != 0) {
        *odd = 1;
#pragma unroll 1
        for (int k = 0; k < kPieces; k++)
            take_out<T>(at(k));
    }
}

/* Adds the infinities and NaN among the values of drafted tokens in slots
 * s0 .. s1 - 1 that a row (mask words `seen`) sees to its outputs of dims
 * d0 .. d0 + 31, in 16-byte pieces that lie swizzled by the row. */
template <typename T>
__device__ __noinline__ void add_odd_values(const PagedTree &a, const TreeItem &x, const uint32_t *seen, int s0, int s1, int d0,
                                            float4 *out, int row) {
    const PagedPool &p = a.p;
    for (int s = s0; s < s1; s++) {
        const int node = s - x.span.prefix, page = lookup(p, x.sequence, s / p.page_size);
        if (page < 0 || !((seen[node >> 5] >> (node & 31)) & 1))
            continue;
        const T *v = static_cast<const T *>(p.values) + int64_t(page) * p.page_stride + int64_t(x.head) * p.head_stride +
                     int64_t(s % p.page_size) * p.slot_stride;
        for (int j = 0; j < 32 && d0 + j < p.head_dim; j++) {
            const float e = to_float(v[d0 + j]);
            if (!(fabsf(e) <= 3.402823466e38f))
                reinterpret_cast<float *>(out + ((j / 4) ^ (row & 7)))[j % 4] += e;
        }
    }
}

constexpr int kNoted = 8;

template <int kStages> struct Shared {
    uint64_t full[kStages], empty[kStages];
    uint64_t queries;                      /* an item's are in shared memory */
    /* of the tiles in each buffer: the softmax may be two tiles ahead of the
     * products, and a barrier tells two phases apart, not three */
    uint64_t logits[2];                    /* a tile's are in tensor memory */
    uint64_t weights[2];                   /* its weights are */
    uint64_t outputs[2];                   /* its product with the values is done */
    uint64_t drained;                      /* products in flight after a wait ran out */
    uint32_t valid[kNoted][2];             /* slots there are of the tiles under way */
    float unit[kRows];                     /* of a row's logits (fp32 queries) */
    uint32_t tmem;
    int dead;                              /* a wait ran out: nothing more is waited for */
    int odd;                               /* an item's value tiles held infinities or NaN */
};

/* Copies of an item of n tiles come in this order: k0 k1 v0 k2 v1 ... */
__device__ __forceinline__ int place_of_keys(int i) { return i == 0 ? 0 : 2 * i - 1; }
__device__ __forceinline__ int place_of_values(int i, int n) { return i == n - 1 ? 2 * i + 1 : 2 * i + 2; }

template <typename T, typename R, typename Plan>
__global__ void __launch_bounds__(kThreads, Plan::kPerSm) tc_kernel(const __grid_constant__ PagedTree a) {
    constexpr int DP = Plan::DP, kStages = Plan::kStages, kTerms = Plan::kTerms, kColumns = Plan::kColumns,
                  kHeld = Plan::kHeld;
    constexpr bool kAside = Plan::kAside;
    constexpr bool kHalf = std::is_same<T, __half>::value;
    constexpr float kSlack = kTerms > 1 ? 0.0f : kHalf ? 7.0f : 8.0f;
    constexpr float kLift = Plan::template lift<T>(); /* log2 of the greatest weight */
    /* sums are freed of it before their logarithm is taken: beside -38 it would lose its last places */
    constexpr float kDrop = power_of_two(-int(kLift));
    extern __shared__ char smem_raw[];
    char *smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    __shared__ Shared<kStages> sh;
    const uint32_t queries_at = smem_u32(smem), ring_at = queries_at + Plan::kQueries;
    const PagedPool &p = a.p;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, D = p.head_dim;
    /* a box of values has all columns of 16 slots where it can */
    const bool wide = a.box >= 16 && a.whole_columns;
    const uint32_t values_lead = wide ? 16 * 128 : kTile * 128, values_step = wide ? kColumns * 16 * 128 : 16 * 128;

    if (tid == 0) {
        for (int i = 0; i < kStages; i++) {
            mbar_init(&sh.full[i], 1);
            mbar_init(&sh.empty[i], 1);
        }
        mbar_init(&sh.queries, kRows);
        mbar_init(&sh.logits[0], 1);
        mbar_init(&sh.logits[1], 1);
        mbar_init(&sh.weights[0], kRows);
        mbar_init(&sh.weights[1], kRows);
        mbar_init(&sh.outputs[0], 1);
        mbar_init(&sh.outputs[1], 1);
        mbar_init(&sh.drained, 1);
        sh.dead = sh.odd = 0;
        fence_barrier_init();
    }
    if (warp == kIssuer) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(&sh.tmem)),
                     "n"(Plan::kMemory)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
    if (warp == kProducer && lane < 2)
        asm volatile("prefetch.tensormap [%0];\n" ::"l"(lane == 0 ? &a.key_map : wide ? &a.wide_value_map : &a.value_map) : "memory");
    tc_before();
    begin_kernel();
    int share;
    TreeCursor cursor = tree_share<kThreads>(a, kTile, kRows, share); /* synchronises the block */
    tc_after();
    const uint32_t tmem = sh.tmem;
    const int start = cursor.pos;

    /* Waits for a barrier's phase.  After kTreeWaitNs somewhere nobody waits
     * any more: the roles run through their steps without doing them. */
    const auto await = [&](uint64_t *bar, uint32_t parity) {
        uint64_t began = 0;
        for (int i = 0;; i++) {
            if (mbar_try_wait(bar, parity))
                return true;
            if ((i & 63) == 63) {
                if (*reinterpret_cast<volatile int *>(&sh.dead))
                    return false;
                const uint64_t now = global_ns();
                if (began == 0) {
                    began = now;
                } else if (now - began > kTreeWaitNs) {
                    *reinterpret_cast<volatile int *>(&sh.dead) = 1;
                    paged_fail(p, kPagedTimeout);
                    return false;
                }
            }
        }
    };
    const auto stage_of = [](uint32_t place) { return place % kStages; };
    const auto parity_of = [](uint32_t place) { return (place / kStages) & 1; };

    TreeItem x;
    uint32_t base = 0; /* copies of earlier items */
    bool alive = true;
    if (warp == kProducer) {
        const int box = a.box, boxes = kTile / box;
        constexpr int kEach = kTile / 32; /* boxes of one slot are so many a lane */
        const int each = boxes > 32 ? boxes / 32 : 1;
        const int ahead = boxes > 32 ? 1 : 32 / boxes;      /* tiles of a look-up */
        const int my_tile = boxes > 32 ? 0 : lane / boxes, my_box = boxes > 32 ? lane * each : lane - my_tile * boxes;
        uint32_t issued = 0;
        while (cursor.next(a, kTile, kRows, x)) {
            const int n = x.tile1 - x.tile0;
            /* pages of the tiles from `looked` on, and of the ones after them */
            int now[kEach], then[kEach], looked = -2 * ahead;
#pragma unroll
            for (int k = 0; k < kEach; k++)
                then[k] = -1;
#pragma unroll 1
            for (int step = 0; step < 2 * n; step++) {
                const bool values = step > 0 && (step % 2 == 0 || step == 2 * n - 1);
                const int i = values ? (step == 2 * n - 1 ? n - 1 : step / 2 - 1) : (step + 1) / 2;
                while (!values && i >= looked + 2 * ahead) { /* keys of a tile that was not looked up */
                    looked += ahead;
#pragma unroll
                    for (int k = 0; k < kEach; k++) {
                        now[k] = then[k];
                        then[k] = -1;
                        const int tile = looked + ahead + my_tile;
                        const int slot = (x.tile0 + tile) * kTile + (my_box + k) * box;
                        if (k < each && tile < n && slot < x.span.length) {
                            const int j = int((uint64_t(unsigned(slot)) * a.page_magic) >> a.page_shift);
                            then[k] = checked_page(p, x.sequence, j);
                        }
                    }
                }
                const uint32_t place = base + step;
                const int stage = stage_of(place);
                if (alive && place >= kStages)
                    alive = __all_sync(0xffffffffu, await(&sh.empty[stage], parity_of(place) ^ 1));
                if (!alive)
                    continue;
                const bool later = i - looked >= ahead;
                const bool mine = my_tile == i - looked - (later ? ahead : 0);
                const int t0 = (x.tile0 + i) * kTile;
                int page[kEach], many = 0;
#pragma unroll
                for (int k = 0; k < kEach; k++) {
                    page[k] = mine ? later ? then[k] : now[k] : -1;
                    many += page[k] >= 0;
                }
                const int all = __reduce_add_sync(0xffffffffu, many);
                if (!values) {
                    const bool full = all == boxes && t0 + kTile <= x.span.length;
#pragma unroll 1
                    for (int w = 0; w < kTile / 32; w++) {
                        uint32_t bits = full ? ~0u : 0u;
                        if (!full) {
#pragma unroll
                            for (int k = 0; k < kEach; k++) {
                                /* the box's slots that there are, as they lie in this word */
                                const int from = (my_box + k) * box - 32 * w;
                                const int to = min(from + box, x.span.length - t0 - 32 * w);
                                if (page[k] >= 0 && from < 32 && to > 0 && to > from)
                                    bits |= (to >= 32 ? ~0u : (1u << to) - 1u) & (from <= 0 ? ~0u : ~0u << from);
                            }
                            bits = __reduce_or_sync(0xffffffffu, bits);
                        }
                        if (lane == 0)
                            sh.valid[(base / 2 + i) % kNoted][w] = bits;
                    }
                }
                if (lane == 0)
                    mbar_expect_tx(&sh.full[stage], uint32_t(all) * box * 128 * kColumns);
                __syncwarp();
                const uint32_t to = ring_at + stage * Plan::kStage, bar = smem_u32(&sh.full[stage]);
#pragma unroll
                for (int k = 0; k < kEach; k++)
                    if (page[k] >= 0) {
                        const int in_tile = (my_box + k) * box, slot = t0 + in_tile;
                        const int y = slot - int((uint64_t(unsigned(slot)) * a.page_magic) >> a.page_shift) * p.page_size;
                        if (values && wide) {
#pragma unroll 1
                            for (int t = 0; t < box; t += 16)
                                copy_box(to + (in_tile + t) * kColumns * 128, &a.wide_value_map, 0, y + t, 0, x.head, page[k], bar);
                        } else {
#pragma unroll
                            for (int c = 0; c < kColumns; c++)
                                copy_box(to + c * kTile * 128 + in_tile * 128, values ? &a.value_map : &a.key_map,
                                         a.whole_columns ? 0 : c * 64, y, a.whole_columns ? c : 0, x.head, page[k], bar);
                        }
                    }
                issued = place + 1;
            }
            base += 2 * n;
        }
        /* what was issued has arrived before the block ends */
        if (!alive)
            for (uint32_t place = issued > kStages ? issued - kStages : 0; place < issued; place++) {
                const uint64_t began = global_ns();
                while (!mbar_try_wait(&sh.full[stage_of(place)], parity_of(place)) && global_ns() - began < kTreeWaitNs)
                    ;
            }
    } else if (warp == kIssuer) {
        if (lane == 0) {
            constexpr uint32_t kShapeS = shape_of<T>(kTile, false), kShapeO = shape_of<T>(DP, true);
            uint32_t items = 0, tiles = 0; /* of the items before */
            /* logits of tile i of the item, from its keys */
            const auto logits = [&](int i) {
                const uint32_t place = base + place_of_keys(i), buffer = (tiles + i) % kBuffers;
                if (alive)
                    alive = await(&sh.full[stage_of(place)], parity_of(place));
                if (!alive)
                    return;
                tc_after();
                const uint64_t k = matrix_at(ring_at + stage_of(place) * Plan::kStage, 16, 1024);
                const uint64_t q = matrix_at(queries_at, 16, 1024);
#pragma unroll
                for (int t = kTerms - 1; t >= 0; t--) /* the small ones first */
#pragma unroll
                    for (int s = 0; s < DP / 16; s++)
                        mma_ss(tmem + buffer * kTile,
                               q + ((t * Plan::kQueryBytes + s / 4 * (kRows * 128) + s % 4 * 32) >> 4),
                               k + ((s / 4 * (kTile * 128) + s % 4 * 32) >> 4), kShapeS, t < kTerms - 1 || s > 0);
                tc_commit(&sh.logits[buffer]);
                tc_commit(&sh.empty[stage_of(place)]);
            };
            while (cursor.next(a, kTile, kRows, x)) {
                const int n = x.tile1 - x.tile0;
                if (alive)
                    alive = await(&sh.queries, items & 1);
                items++;
                /* logits run ahead of the weights by kBuffers tiles */
#pragma unroll 1
                for (int i = -kBuffers; i < n; i++) {
                    if (i >= 0) {
                        const uint32_t place = base + place_of_values(i, n), buffer = (tiles + i) % kBuffers;
                        if (alive)
                            alive = await(&sh.full[stage_of(place)], parity_of(place)) &&
                                    await(&sh.weights[buffer], (tiles + i) / kBuffers & 1);
                        if (alive) {
                            tc_after();
                            const uint64_t v = matrix_at(ring_at + stage_of(place) * Plan::kStage, values_lead, 1024);
                            const uint32_t weights = tmem + buffer * kTile;
#pragma unroll
                            for (int t = kTerms - 1; t >= 0; t--)
#pragma unroll
                                for (int s = 0; s < kTile / 16; s++)
                                    mma_ts(tmem + Plan::kOutputs, (t < 2 ? weights + t * (kTile / 2) : tmem + Plan::kThird) + s * 8,
                                           v + s * (values_step >> 4), kShapeO, (!kAside && i > 0) || t < kTerms - 1 || s > 0);
                            tc_commit(&sh.outputs[buffer]);
                            tc_commit(&sh.empty[stage_of(place)]);
                        }
                    }
                    if (i + kBuffers < n)
                        logits(i + kBuffers);
                }
                base += 2 * n;
                tiles += n;
            }
            if (!alive) { /* products in flight end before tensor memory is given back */
                tc_commit(&sh.drained);
                const uint64_t began = global_ns();
                while (!mbar_try_wait(&sh.drained, 0) && global_ns() - began < kTreeWaitNs)
                    ;
            }
        }
        __syncwarp();
    } else {
        const uint32_t lanes = uint32_t(warp * 32) << 16, outputs_at = tmem + lanes + Plan::kOutputs,
                       sums_at = tmem + lanes + Plan::kSums;
        const auto everyone = [] { named_barrier(1, kRows); };
        /* A barrier for every buffer: no phase of one is waited for when the next may
         * have ended too, or have not begun. */
        const auto await_outputs = [&](uint32_t tile) { return await(&sh.outputs[tile % kBuffers], tile / kBuffers & 1); };
        uint32_t tiles = 0; /* of the items before */
        int4 join = make_int4(0, 0, 0, 0);
        tree_blind_rows<R>(a, tid, kRows);
        while (cursor.next(a, kTile, kRows, x)) {
            const int n = x.tile1 - x.tile0;
            const bool counts = tid < x.rows;
            const bool idle = warp * 32 >= x.rows; /* a warp without rows */
            const uint32_t *seen = a.mask;
            if (counts)
                seen += (int64_t(x.span.row0) + tree_node(a, x.first_row + tid)) * a.mask_words;
            const uint32_t seen0 = counts ? seen[0] : 0u; /* most trees have no more words */

            /* the queries: a row's DP / 8 pieces of 8 dims by neighbouring lanes,
             * kBatch of them in flight a thread */
            constexpr int kAcross = DP / 8, kStep = kRows / kAcross, kBatch = kTerms == 1 ? kRows / kStep : 8;
            constexpr int kLoads = sizeof(R) / 2; /* of 16 bytes a piece */
            static_assert(kRows % (kBatch * kStep) == 0, "whole batches");
            const int c = tid % kAcross;
            /* a scale below 0 turns the queries round */
            const uint32_t flip = a.scale < 0.0f ? (sizeof(R) == 4 ? 0x80000000u : 0x80008000u) : 0u;
#pragma unroll 1
            for (int r0 = tid / kAcross; r0 < (x.rows + kAcross - 1) / kAcross * kAcross; r0 += kBatch * kStep) {
                uint4 pieces[kBatch][kLoads];
#pragma unroll
                for (int k = 0; k < kBatch; k++) {
                    const int r = r0 + k * kStep;
#pragma unroll
                    for (int j = 0; j < kLoads; j++)
                        pieces[k][j] = make_uint4(0, 0, 0, 0);
                    if (r < x.rows && c * 8 < D) {
                        int64_t q_row;
                        int h;
                        tree_row(a, x.span.row0, x.head, x.first_row + r, q_row, h);
                        const R *q = static_cast<const R *>(a.q) + q_row * a.q_stride + h * D + c * 8;
#pragma unroll
                        for (int j = 0; j < kLoads; j++)
                            pieces[k][j] = a.aligned ? *reinterpret_cast<const uint4 *>(q + j * (8 / kLoads))
                                                     : load_elements(q + j * (8 / kLoads));
                    }
                }
#pragma unroll
                for (int k = 0; k < kBatch; k++) {
                    const int r = r0 + k * kStep;
                    char *to = smem + (c >> 3) * (kRows * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4);
#pragma unroll
                    for (int j = 0; j < kLoads; j++) {
                        pieces[k][j].x ^= flip;
                        pieces[k][j].y ^= flip;
                        pieces[k][j].z ^= flip;
                        pieces[k][j].w ^= flip;
                    }
                    if constexpr (kTerms == 1) {
                        *reinterpret_cast<uint4 *>(to) = pieces[k][0];
                    } else {
                        float v[8] = {
                            __uint_as_float(pieces[k][0].x), __uint_as_float(pieces[k][0].y), __uint_as_float(pieces[k][0].z),
                            __uint_as_float(pieces[k][0].w), __uint_as_float(pieces[k][kLoads - 1].x),
                            __uint_as_float(pieces[k][kLoads - 1].y), __uint_as_float(pieces[k][kLoads - 1].z),
                            __uint_as_float(pieces[k][kLoads - 1].w)};
                        float unit = fabsf(a.scale) * kTreeLog2e;
                        if constexpr (kHalf) { /* greatest |q| to [2^10, 2^11) */
                            float top = 0.0f;
#pragma unroll
                            for (int j = 0; j < 8; j++)
                                top = fmaxf(top, fabsf(v[j]));
#pragma unroll
                            for (int e = kAcross / 2; e > 0; e >>= 1)
                                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, e));
                            const int e = int(__float_as_uint(top) >> 23);
                            if (e > 0 && e < 255) {
                                const int field = min(264 - e, 253);
                                const float gain = __uint_as_float(uint32_t(field) << 23);
#pragma unroll
                                for (int j = 0; j < 8; j++)
                                    v[j] *= gain;
                                /* not 0, which would make NaN of a masked -infinity; at 2^-126 no
                                 * logit is above 2^-90, and weights are as at any unit below */
                                unit = fmaxf(unit * __uint_as_float(uint32_t(254 - field) << 23), 1.17549435e-38f);
                            }
                        }
                        if (c == 0)
                            sh.unit[r] = unit;
#pragma unroll
                        for (int t = 0; t < kTerms; t++) {
                            uint32_t e[4];
#pragma unroll
                            for (int j = 0; j < 4; j++) {
                                e[j] = Pair<T>::pack(v[2 * j], v[2 * j + 1]);
                                const float2 taken = Pair<T>::unpack(e[j]);
                                v[2 * j] -= taken.x;
                                v[2 * j + 1] -= taken.y;
                            }
                            *reinterpret_cast<uint4 *>(to + t * Plan::kQueryBytes) = make_uint4(e[0], e[1], e[2], e[3]);
                        }
                    }
                }
            }
            fence_async();
            mbar_arrive(&sh.queries);
            if constexpr (kTerms > 1)
                everyone(); /* the units */

            const float unit = kTerms > 1 ? sh.unit[tid] : fabsf(a.scale) * kTreeLog2e;
            /* weights are 2^((s - m) unit + kLift), m a maximum of s.  (Differences of s: beside products
             * s unit of 2^27 and more, rounded, the greatest weight would be off by their last place.) */
            float m = -INFINITY, l = 0.0f;
            /* kAside: O is a tile's own; earlier tiles' sum is put aside, to be multiplied by `ratio` */
            float ratio = 1.0f, held[kHeld > 0 ? kHeld : 1];
#pragma unroll
            for (int j = 0; j < kHeld; j++)
                held[j] = 0.0f;
            const auto add_sums = [&](int c, float *o, bool there) {
                if (c >= DP - kHeld) {
#pragma unroll
                    for (int j = 0; j < kHeld; j++)
                        o[j] = fmaf(held[j], ratio, o[j]);
                } else if (there) {
                    float sums[32];
                    tmem_load32(sums_at + c, sums);
                    tc_wait_ld();
#pragma unroll
                    for (int j = 0; j < 32; j++)
                        o[j] = fmaf(sums[j], ratio, o[j]);
                }
            };
#pragma unroll 1
            for (int i = 0; i < n; i++, tiles++) {
                const uint32_t logits_at = tmem + lanes + tiles % kBuffers * kTile;
                const int t0 = (x.tile0 + i) * kTile;
                if (alive)
                    alive = await(&sh.logits[tiles % kBuffers], tiles / kBuffers & 1);
                alive = __all_sync(0xffffffffu, alive);
                if (!alive)
                    continue;
                tc_after();
                const volatile uint32_t *noted = sh.valid[(base / 2 + i) % kNoted];
                uint32_t words[2] = {noted[0], noted[1]};
                const bool plain = t0 + kTile <= x.span.prefix && (words[0] & words[1]) == ~0u;
                if (!plain) {
                    /* values that must not meet weights of 0 */
                    const uint32_t place = base + place_of_values(i, n);
                    alive = __all_sync(0xffffffffu, await(&sh.full[stage_of(place)], parity_of(place)));
                    static_assert(kRows == 2 * kTile, "two threads a slot");
                    const int slot = tid >> 1;
                    const bool there = (noted[slot >> 5] >> (slot & 31)) & 1;
                    if (alive && (!there || t0 + slot >= x.span.prefix))
                        clean_values<T, DP>(ring_at + stage_of(place) * Plan::kStage + (slot >> 4) * values_step + (slot & 15) * 128,
                                            slot, tid & 1, values_lead, there, &sh.odd);
                    fence_async();
                }
                if (kAside && i > 0 && !idle && alive) {
                    alive = __all_sync(0xffffffffu, await_outputs(tiles - 1));
                    tc_after();
                    if (alive) {
#pragma unroll 1
                        for (int c = 0; c < DP - kHeld; c += 32) {
                            float o[32];
                            tmem_load32(outputs_at + c, o);
                            tc_wait_ld();
                            add_sums(c, o, i > 1);
                            tmem_store32(sums_at + c, o);
                        }
                        if constexpr (kHeld > 0) {
                            static_assert(kHeld <= 32, "one piece");
                            float o[32];
                            tmem_load32(outputs_at + DP - kHeld, o);
                            tc_wait_ld();
                            add_sums(DP - kHeld, o, true);
#pragma unroll
                            for (int j = 0; j < kHeld; j++)
                                held[j] = o[j];
                        }
                        ratio = 1.0f;
                    }
                }
                if (!idle && alive) {
                    float s[kTile];
                    tmem_load32(logits_at, s);
                    tmem_load32(logits_at + 32, s + 32);
                    tc_wait_ld();
                    if (!plain)
#pragma unroll
                        for (int k = 0; k < kTile; k += 32) {
                            uint32_t sees = words[k / 32];
                            const int node = t0 + k - x.span.prefix;
                            if (node > -32)
                                sees &= x.span.n <= 32 ? tree_sees(&seen0, node, x.span.n) : tree_sees(seen, node, x.span.n);
#pragma unroll
                            for (int j = 0; j < 32; j++)
                                s[k + j] = (sees >> j) & 1 ? s[k + j] : -INFINITY;
                        }
                    float top = s[0], other = s[1];
#pragma unroll
                    for (int k = 2; k < kTile; k += 2) {
                        top = fmaxf(top, s[k]);
                        other = fmaxf(other, s[k + 1]);
                    }
                    top = fmaxf(top, other);
                    const float next = (top - m) * unit > kSlack ? top : m; /* (NaN: both are -infinity) */
                    if (__any_sync(0xffffffffu, next != m)) {
                        const float keep = m == next ? 1.0f : power2((m - next) * unit);
                        l *= keep;
                        m = next;
                        ratio *= keep;
                        if (!kAside && i > 0) { /* once the products before are complete */
                            alive = __all_sync(0xffffffffu, await_outputs(tiles - 1));
                            tc_after();
#pragma unroll 1
                            for (int c = 0; c < DP && alive; c += 32) {
                                float o[32];
                                tmem_load32(outputs_at + c, o);
                                tc_wait_ld();
#pragma unroll
                                for (int j = 0; j < 32; j++)
                                    o[j] *= keep;
                                tmem_store32(outputs_at + c, o);
                            }
                        }
                    }
                    const float none = m == -INFINITY ? 0.0f : -m;
                    const Two less = two_of(none, none), units = two_of(unit, unit),
                              lift = kHalf ? two_of(kLift, kLift) : two_of(1.0f / kDrop, 1.0f / kDrop);
                    float sum = 0.0f, sum1 = 0.0f;
#pragma unroll
                    for (int k = 0; k < kTile; k += 32) {
                        uint32_t e[kTerms][16];
#pragma unroll
                        for (int j = 0; j < 16; j++) {
                            Two z = two_of(s[k + 2 * j], s[k + 2 * j + 1]);
                            asm("add.rn.f32x2 %0, %0, %1;\n" : "+l"(z) : "l"(less));
                            float w0, w1;
                            if constexpr (kHalf) {
                                asm("fma.rn.f32x2 %0, %0, %1, %2;\n" : "+l"(z) : "l"(units), "l"(lift));
                                w0 = power2(parts_of(z).x);
                                w1 = power2(parts_of(z).y);
                            } else { /* beside -38 the exponent would lose its last 5 bits */
                                asm("mul.rn.f32x2 %0, %0, %1;\n" : "+l"(z) : "l"(units));
                                z = two_of(power2(parts_of(z).x), power2(parts_of(z).y));
                                asm("mul.rn.f32x2 %0, %0, %1;\n" : "+l"(z) : "l"(lift));
                                w0 = parts_of(z).x;
                                w1 = parts_of(z).y;
                            }
                            sum += w0;
                            sum1 += w1;
#pragma unroll
                            for (int t = 0; t < kTerms; t++) {
                                e[t][j] = Pair<T>::pack(w0, w1);
                                if (t + 1 < kTerms) {
                                    const float2 taken = Pair<T>::unpack(e[t][j]);
                                    w0 -= taken.x;
                                    w1 -= taken.y;
                                }
                            }
                        }
#pragma unroll
                        for (int t = 0; t < kTerms; t++)
                            tmem_store16((t < 2 ? logits_at + t * (kTile / 2) : tmem + lanes + Plan::kThird) + k / 2, e[t]);
                    }
                    l += sum + sum1;
                    tc_wait_st();
                }
                tc_before();
                mbar_arrive(&sh.weights[tiles % kBuffers]);
            }
            base += 2 * n;

            /* the end of the item, or of this block's part of it */
            if (alive && n > 1) /* the products may be two tiles behind */
                alive = await_outputs(tiles - 2);
            if (alive)
                alive = await_outputs(tiles - 1);
            alive = __all_sync(0xffffffffu, alive);
            tc_after();
            everyone(); /* all products are done: the queries' place is free */
            const bool odd = sh.odd != 0, whole = x.whole();
            const float factor = !whole ? 1.0f : l == 0.0f ? 0.0f : 1.0f / l;
            const TreePart part = tree_part(a, blockIdx.x, x.first <= start ? 0 : 1, x.rows);
            if (counts && alive) {
                if (!whole) {
                    const float most = m * unit;
                    part.maxima[tid] = most;
                    part.rests[tid] = fabsf(most) < INFINITY ? fmaf(m, unit, -most) : 0.0f;
                    part.sums[tid] = l;
                } else if (a.lse) {
                    int64_t out_row;
                    int h;
                    tree_row(a, x.span.row0, x.head, x.first_row + tid, out_row, h);
                    a.lse[out_row * p.heads + h] = l == 0.0f ? -INFINITY : fmaf(m, unit, log2f(l * kDrop)) * kTreeLn2;
                }
            }
            /* 32 dims at a time leave through a warp's 4 KB of the queries'
             * place, 128 bytes of a row by 8 lanes */
            const int piece = lane & 7;
            float4 *rows_at = reinterpret_cast<float4 *>(smem + warp * 32 * 128);
            char *to[8]; /* row 4 i + lane / 8 of the warp, from this lane's dims on */
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int r = warp * 32 + i * 4 + (lane >> 3);
                if (whole) {
                    int64_t out_row;
                    int h;
                    tree_row(a, x.span.row0, x.head, x.first_row + r, out_row, h);
                    to[i] = reinterpret_cast<char *>(static_cast<R *>(a.out) + out_row * a.out_stride + h * D + piece * 4);
                } else {
                    to[i] = reinterpret_cast<char *>(part.out + r * D + piece * 4);
                }
            }
            const int mine_from = warp * 32 + (lane >> 3);
#pragma unroll 1
            for (int d0 = 0; d0 < D && !idle && alive; d0 += 32) {
                float o[32];
                tmem_load32(outputs_at + d0, o);
                tc_wait_ld();
                if constexpr (kAside)
                    if (n > 1)
                        add_sums(d0, o, true);
                __syncwarp();
                float4 *mine = rows_at + lane * 8;
#pragma unroll
                for (int j = 0; j < 8; j++)
                    mine[j ^ (lane & 7)] = make_float4(o[4 * j] * factor, o[4 * j + 1] * factor, o[4 * j + 2] * factor,
                                                       o[4 * j + 3] * factor);
                if (odd && counts)
                    add_odd_values<T>(a, x, seen, max(x.span.prefix, x.tile0 * kTile), min(x.span.length, x.tile1 * kTile), d0, mine,
                                      lane);
                __syncwarp();
                float4 v[8];
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const int r = i * 4 + (lane >> 3);
                    v[i] = rows_at[r * 8 + (piece ^ (r & 7))];
                }
                const int rows = d0 + piece * 4 < D ? x.rows : 0; /* that have these dims */
                if (!whole || sizeof(R) == 4) {
                    if (!whole || a.aligned) {
#pragma unroll
                        for (int i = 0; i < 8; i++)
                            if (mine_from + i * 4 < rows)
                                *reinterpret_cast<float4 *>(to[i] + d0 * 4) = v[i];
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; i++)
                            store_elements(reinterpret_cast<float *>(to[i]) + d0, v[i], mine_from + i * 4 < rows);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        R *at = reinterpret_cast<R *>(to[i]) + d0;
                        if (!a.aligned)
                            store_elements(at, v[i], mine_from + i * 4 < rows);
                        else if (mine_from + i * 4 < rows)
                            *reinterpret_cast<uint2 *>(at) = make_uint2(pack_outputs<R>(v[i].x, v[i].y), pack_outputs<R>(v[i].z, v[i].w));
                    }
                }
            }
            if (!whole && x.tile0 == 0)
                join = tree_join(x, share);
            tc_before();
            everyone(); /* the queries' place is free again */
            if (tid == 0)
                sh.odd = 0;
        }
        if (tid == 0)
            a.joins[blockIdx.x] = join;
    }
    tc_before();
    __syncthreads();
    if (warp == kIssuer) {
        tc_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "n"(Plan::kMemory) : "memory");
    }
}

template <typename T, typename R, int DP, int kTerms> cudaError_t launch(const PagedTree &a, cudaStream_t s) {
    using Plan = TcPlan<DP, kTerms>;
    const auto kernel = tc_kernel<T, R, Plan>;
    static bool set[kMaxDevices] = {};
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess)
        return e;
    if (!set[device % kMaxDevices]) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Plan::kBytes);
        if (e != cudaSuccess)
            return e;
        set[device % kMaxDevices] = true;
    }
    const int ctas = a.sms * Plan::kPerSm;
    e = launch_kernel(kernel, dim3(ctas), kThreads, Plan::kBytes, s, 1, a);
    return e != cudaSuccess ? e : tree_join_parts(a, ctas, kRows, power_of_two(-int(Plan::template lift<T>())), s);
}

template <typename T, int DP> cudaError_t launch(const PagedTree &a, cudaStream_t s) {
    return a.type == 0 ? launch<T, float, DP, std::is_same<T, __half>::value ? 2 : 3>(a, s) : launch<T, T, DP, 1>(a, s);
}

} // namespace

cudaError_t paged_tree_tc(const PagedTree &a, cudaStream_t s) {
    if (a.p.type == 1)
        return a.p.head_dim <= 64 ? launch<__half, 64>(a, s) : launch<__half, 128>(a, s);
    return a.p.head_dim <= 64 ? launch<__nv_bfloat16, 64>(a, s) : launch<__nv_bfloat16, 128>(a, s);
}

} // namespace nut
