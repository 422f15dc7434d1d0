/* Attention of drafted tokens over a 16-bit paged KV cache on the tensor cores
 * (nut_paged_tree_attention, head_dim up to 128).
 *
 * All rows of a sequence that share a kv head (drafted tokens by query heads)
 * are one matrix, so a pass over the cache serves them together: logits
 * S = Q K^T and outputs O += P V of 128 rows by tcgen05.mma, with S, P and O in
 * tensor memory and a thread for each row in the softmax between them.
 *
 *   warp 8      copies key and value tiles (TMA boxes of a page's slots) into
 *               a ring of stages, and notes which slots there are
 *   warp 9      issues the products
 *   warps 0-3, 4-7   the softmax of two streams, each with its own S, P and O:
 *               the halves of more than 128 rows on the same tiles, else
 *               every other tile of the same rows, joined at the item's end.
 *               While one stream does its softmax the other's products run.
 *
 * Queries in fp32 are split into 16-bit terms that multiply the same keys, and
 * so are their weights: two for fp16 (queries first scaled by a power of two
 * to [2^10, 2^11)), three for bf16.  Weights are kept in the 16-bit type's
 * range by a power of two: of fp16 the greatest is 2^8 to 2^15, since fp16 ends
 * at 2^-24; of bf16 it is 2^-30 at most, so that no sum of values near bf16's
 * greatest overflows.  A row's maximum may lag behind by kSlack: its outputs
 * are rescaled only when it rises by more.
 *
 * Values of slots that some rows do not see would meet weights of 0 in the
 * product: among the drafted tokens infinities and NaN are taken out of the
 * tile, and added at the end to the rows that see them.
 */
#include <cstdint>
#include <type_traits>
#include <cuda_runtime.h>

#include "paged_tree.cuh"
#include "stream.cuh"

namespace nut {
namespace {

constexpr int kStreams = 2;
constexpr int kThreads = kStreams * 128 + 64;
constexpr int kProducer = kStreams * 4, kIssuer = kProducer + 1; /* warps */
constexpr uint64_t kTreeWaitNs = 2000000000ull;

/* kTerms: 16-bit terms of a query and of a weight. */
template <int DP_, int kTerms_> struct TcPlan {
    static constexpr int DP = DP_, kTerms = kTerms_;
    /* three terms of 128 weights do not fit in their logits' place */
    static constexpr int kTile = kTerms == 3 ? 64 : 128;
    static constexpr int kColumns = DP / 64; /* of 128 bytes */
    static constexpr int kQueryTiles = kTerms == 1 ? 2 : 1;
    static constexpr int kBlockRows = 128 * kQueryTiles;
    static constexpr int kQueryBytes = 128 * DP * 2;
    static constexpr int kQueries = kQueryBytes * kQueryTiles * kTerms;
    static constexpr int kStage = kTile * DP * 2;
    static constexpr int kFit = (227 * 1024 - 1024 - 4096 - kQueries) / kStage; /* beside alignment and static shared memory */
    static constexpr int kStages = kFit < 10 ? kFit : 10;
    static constexpr int kBytes = 1024 + kQueries + kStages * kStage;
    /* tensor memory: S (P in its place) of both streams, then O of both */
    static constexpr int kLogits = kTile > kTerms * kTile / 2 ? kTile : kTerms * kTile / 2;
    static constexpr int kOutputs = kStreams * kLogits;
    static_assert(kOutputs + kStreams * DP <= 512, "columns of tensor memory");
    static_assert(kQueries >= 128 * DP * 4, "the streams' outputs meet there");
    static_assert(kStages >= 4, "keys of two tiles and values of one are in use at a time");
};

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

/* A matrix in 128-byte rows with the 128-byte swizzle, 1024 bytes to 8 rows.
 * Rows along the product's M or N (K-major): `lead` has no meaning.  Rows
 * along its K (MN-major): 8 of K are 1024 bytes, 64 of N are `lead`. */
__device__ __forceinline__ uint64_t matrix_at(uint32_t addr, uint32_t lead) {
    return uint64_t((addr >> 4) & 0x3fffu) | uint64_t((lead >> 4) & 0x3fffu) << 16 | uint64_t(1024 >> 4) << 32 |
           uint64_t(1) << 46 | uint64_t(2) << 61;
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
};

/* ---- the kernel ---------------------------------------------------------- */

template <int kStages> struct Shared {
    uint64_t full[kStages], empty[kStages];
    uint64_t queries;                      /* an item's are in shared memory */
    uint64_t logits[kStreams];             /* a tile's are in tensor memory */
    uint64_t weights[kStreams];            /* and its weights */
    uint64_t outputs[kStreams], drained;
    uint32_t valid[kStages][4];            /* slots there are of a value tile */
    float unit[128];                       /* of a row's logits (fp32 queries) */
    float maxima[kStreams][128], sums[kStreams][128];
    uint32_t tmem;
    int dead;                              /* a wait ran out: nothing more is waited for */
    int odd;                               /* an item's value tiles held infinities or NaN */
};

/* Where a tile's keys and values lie in the order of copies of an item of n
 * tiles: k0 k1 v0 k2 v1 ... */
__device__ __forceinline__ int place_of_keys(int i) { return i == 0 ? 0 : 2 * i - 1; }
__device__ __forceinline__ int place_of_values(int i, int n) { return i == n - 1 ? 2 * i + 1 : 2 * i + 2; }

template <typename T, typename R, typename Plan>
__global__ void __launch_bounds__(kThreads, 1) tc_kernel(const __grid_constant__ PagedTree a) {
    constexpr int DP = Plan::DP, kTile = Plan::kTile, kStages = Plan::kStages, kTerms = Plan::kTerms,
                  kColumns = Plan::kColumns;
    constexpr bool kHalf = std::is_same<T, __half>::value;
    constexpr float kSlack = kTerms > 1 ? 0.0f : kHalf ? 7.0f : 8.0f;
    constexpr float kLift = !kHalf ? -38.0f : kTerms > 1 ? 15.0f : 8.0f; /* log2 of the greatest weight */
    extern __shared__ char smem_raw[];
    char *smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    __shared__ Shared<kStages> sh;
    const uint32_t queries_at = smem_u32(smem), ring_at = queries_at + Plan::kQueries;
    const PagedPool &p = a.p;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, D = p.head_dim;

    if (tid == 0) {
        for (int i = 0; i < kStages; i++) {
            mbar_init(&sh.full[i], 1);
            mbar_init(&sh.empty[i], 1);
        }
        mbar_init(&sh.queries, kStreams * 128);
        for (int w = 0; w < kStreams; w++) {
            mbar_init(&sh.logits[w], 1);
            mbar_init(&sh.weights[w], 128);
            mbar_init(&sh.outputs[w], 1);
        }
        mbar_init(&sh.drained, 1); /* products in flight after a wait ran out */
        sh.dead = sh.odd = 0;
        fence_barrier_init();
    }
    if (warp == kIssuer) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;\n" ::"r"(smem_u32(&sh.tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
    tc_before();
    begin_kernel();
    int share;
    TreeCursor cursor = tree_share<kThreads>(a, kTile, Plan::kBlockRows, share); /* synchronises the block */
    tc_after();
    const uint32_t tmem = sh.tmem;
    const int start = cursor.pos;
    tree_blind_rows<R>(a);

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
        const int each = boxes > 32 ? boxes / 32 : 1;       /* boxes of a lane */
        const int ahead = boxes > 32 ? 1 : 32 / boxes;      /* tiles of a look-up */
        const int my_tile = boxes > 32 ? 0 : lane / boxes, my_box = boxes > 32 ? lane * each : lane - my_tile * boxes;
        uint32_t issued = 0;
        while (cursor.next(a, kTile, Plan::kBlockRows, x)) {
            const int n = x.tile1 - x.tile0;
            /* pages of the tiles from `looked` on, and of the ones after them */
            int now[4], then[4], looked = -1;
            const auto look = [&](int i, int (&page)[4]) {
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    page[k] = -1;
                    const int slot = (x.tile0 + i + my_tile) * kTile + (my_box + k) * box;
                    if (k < each && i + my_tile < n && slot < x.span.length) {
                        const int j = int((uint64_t(unsigned(slot)) * a.page_magic) >> a.page_shift);
                        page[k] = checked_page(p, x.sequence, j);
                    }
                }
            };
            /* copies tile i's keys or values */
            const auto copy = [&](int i, bool values, const int (&page)[4], int offset) {
                const uint32_t place = base + (values ? place_of_values(i, n) : place_of_keys(i));
                const int stage = stage_of(place);
                if (alive && place >= kStages)
                    alive = __all_sync(0xffffffffu, await(&sh.empty[stage], parity_of(place) ^ 1));
                if (!alive)
                    return;
                const bool mine = my_tile == offset;
                const int t0 = (x.tile0 + i) * kTile;
                int many = 0;
#pragma unroll
                for (int k = 0; k < 4; k++)
                    many += mine && page[k] >= 0;
                const int all = __reduce_add_sync(0xffffffffu, many);
                if (values) {
                    uint32_t words[kTile / 32];
#pragma unroll
                    for (int w = 0; w < kTile / 32; w++)
                        words[w] = ~0u;
                    if (all < boxes || t0 + kTile > x.span.length) {
#pragma unroll
                        for (int w = 0; w < kTile / 32; w++) {
                            uint32_t bits = 0;
#pragma unroll
                            for (int k = 0; k < 4; k++) {
                                /* the box's slots that there are, as they lie in this word */
                                const int from = (my_box + k) * box - 32 * w;
                                const int to = min(from + box, x.span.length - t0 - 32 * w);
                                if (mine && page[k] >= 0 && from < 32 && to > 0 && to > from)
                                    bits |= (to >= 32 ? ~0u : (1u << to) - 1u) & (from <= 0 ? ~0u : ~0u << from);
                            }
                            words[w] = __reduce_or_sync(0xffffffffu, bits);
                        }
                    }
                    if (lane == 0)
#pragma unroll
                        for (int w = 0; w < kTile / 32; w++)
                            sh.valid[stage][w] = words[w];
                }
                if (lane == 0)
                    mbar_expect_tx(&sh.full[stage], uint32_t(all) * box * 128 * kColumns);
                __syncwarp();
                const uint32_t to = ring_at + stage * Plan::kStage, bar = smem_u32(&sh.full[stage]);
                const CUtensorMap *map = values ? &a.value_map : &a.key_map;
#pragma unroll
                for (int k = 0; k < 4; k++)
                    if (mine && page[k] >= 0) {
                        const int slot = t0 + (my_box + k) * box;
                        const int j = int((uint64_t(unsigned(slot)) * a.page_magic) >> a.page_shift);
                        const int y = slot - j * p.page_size;
#pragma unroll
                        for (int c = 0; c < kColumns; c++)
                            copy_box(to + c * kTile * 128 + (my_box + k) * box * 128, map, a.whole_columns ? 0 : c * 64, y,
                                     a.whole_columns ? c : 0, x.head, page[k], bar);
                    }
                issued = max(issued, place + 1);
            };
            look(0, now);
            looked = 0;
            look(ahead, then);
            copy(0, false, now, 0);
            for (int i = 0; i < n; i++) {
                /* keys of tile i + 1, then values of tile i */
                if (i + 1 < n) {
                    if (i + 1 - looked < ahead)
                        copy(i + 1, false, now, i + 1 - looked);
                    else
                        copy(i + 1, false, then, i + 1 - looked - ahead);
                }
                copy(i, true, now, i - looked);
                if (i + 1 - looked == ahead) {
#pragma unroll
                    for (int k = 0; k < 4; k++)
                        now[k] = then[k];
                    looked += ahead;
                    look(looked + ahead, then);
                }
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
            uint32_t items = 0, turns[kStreams] = {0, 0};
            /* S of a stream = Q K^T */
            const auto logits = [&](int w, int query_tile, uint32_t place) {
                const uint32_t k = ring_at + stage_of(place) * Plan::kStage;
#pragma unroll
                for (int t = 0; t < kTerms; t++) {
                    const uint32_t q = queries_at + (t * Plan::kQueryTiles + query_tile) * Plan::kQueryBytes;
#pragma unroll
                    for (int s = 0; s < DP / 16; s++)
                        mma_ss(tmem + w * Plan::kLogits, matrix_at(q + s / 4 * (128 * 128) + s % 4 * 32, 16),
                               matrix_at(k + s / 4 * (kTile * 128) + s % 4 * 32, 16), kShapeS, t > 0 || s > 0);
                }
            };
            /* O of a stream += P V */
            const auto outputs = [&](int w, uint32_t place, bool first) {
                const uint32_t v = ring_at + stage_of(place) * Plan::kStage;
#pragma unroll
                for (int t = 0; t < kTerms; t++)
#pragma unroll
                    for (int s = 0; s < kTile / 16; s++)
                        mma_ts(tmem + Plan::kOutputs + w * DP, tmem + w * Plan::kLogits + t * (kTile / 2) + s * 8,
                               matrix_at(v + s * 2048, kTile * 128), kShapeO, !first || t > 0 || s > 0);
            };
            const auto arrived = [&](uint32_t place) {
                if (alive)
                    alive = await(&sh.full[stage_of(place)], parity_of(place));
                if (alive)
                    tc_after();
            };
            while (cursor.next(a, kTile, Plan::kBlockRows, x)) {
                const int n = x.tile1 - x.tile0;
                const bool both = x.rows > 128; /* streams take halves of the rows, else every other tile */
                if (alive)
                    alive = await(&sh.queries, items & 1);
                items++;
                if (both) {
                    arrived(base);
                    if (alive)
                        for (int w = 0; w < 2; w++) {
                            logits(w, w % Plan::kQueryTiles, base);
                            tc_commit(&sh.logits[w]);
                        }
                    if (alive)
                        tc_commit(&sh.empty[stage_of(base)]);
                    for (int i = 0; i < n; i++) {
                        const uint32_t values = base + place_of_values(i, n), keys = base + place_of_keys(i + 1);
                        if (i + 1 < n)
                            arrived(keys);
                        arrived(values);
#pragma unroll
                        for (int w = 0; w < 2; w++) {
                            if (alive)
                                alive = await(&sh.weights[w], turns[w] & 1);
                            turns[w]++;
                            if (!alive)
                                continue;
                            tc_after();
                            outputs(w, values, i == 0);
                            if (i + 1 < n) {
                                logits(w, w % Plan::kQueryTiles, keys);
                                tc_commit(&sh.logits[w]);
                            } else {
                                tc_commit(&sh.outputs[w]);
                            }
                        }
                        if (alive) {
                            tc_commit(&sh.empty[stage_of(values)]);
                            if (i + 1 < n)
                                tc_commit(&sh.empty[stage_of(keys)]);
                        }
                    }
                } else {
                    for (int i = 0; i < 2 && i < n; i++) {
                        const uint32_t keys = base + place_of_keys(i);
                        arrived(keys);
                        if (!alive)
                            continue;
                        logits(i, 0, keys);
                        tc_commit(&sh.logits[i]);
                        tc_commit(&sh.empty[stage_of(keys)]);
                    }
                    for (int i = 0; i < n; i++) {
                        const int w = i & 1;
                        const uint32_t values = base + place_of_values(i, n);
                        arrived(values);
                        if (alive)
                            alive = await(&sh.weights[w], turns[w] & 1);
                        turns[w]++;
                        if (alive) {
                            tc_after();
                            outputs(w, values, i < 2);
                            tc_commit(&sh.empty[stage_of(values)]);
                            if (i + 2 >= n)
                                tc_commit(&sh.outputs[w]);
                        }
                        if (i + 2 < n) {
                            const uint32_t keys = base + place_of_keys(i + 2);
                            arrived(keys);
                            if (alive) {
                                logits(w, 0, keys);
                                tc_commit(&sh.logits[w]);
                                tc_commit(&sh.empty[stage_of(keys)]);
                            }
                        }
                    }
                }
                base += 2 * n;
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
        const int w = warp >> 2, row = tid & 127; /* stream, row of the tile */
        const uint32_t lanes = uint32_t((warp & 3) * 32) << 16;
        const uint32_t logits_at = tmem + lanes + w * Plan::kLogits, outputs_at = tmem + lanes + Plan::kOutputs + w * DP;
        const auto everyone = [] { named_barrier(1, kStreams * 128); };
        uint32_t turns = 0, ends = 0;
        int4 join = make_int4(0, 0, 0, 0);
        while (cursor.next(a, kTile, Plan::kBlockRows, x)) {
            const int n = x.tile1 - x.tile0;
            const bool both = x.rows > 128;

            /* the queries: a row's DP / 8 pieces of 8 dims by neighbouring lanes */
            constexpr int kAcross = DP / 8;
            const int query_rows = both ? kStreams * 128 : 128;
            for (int i = tid; i < query_rows * kAcross; i += kStreams * 128) {
                const int r = i / kAcross, c = i % kAcross;
                const bool there = r < x.rows;
                int64_t q_row = 0;
                int h = 0;
                if (there)
                    tree_row(a, x.span.row0, x.head, x.first_row + r, q_row, h);
                const R *q = static_cast<const R *>(a.q) + q_row * a.q_stride + int64_t(h) * D + c * 8;
                char *to = smem + (r >> 7) * Plan::kQueryBytes + (c >> 3) * (128 * 128) + (r & 127) * 128 +
                           (((c & 7) ^ (r & 7)) << 4);
                if constexpr (kTerms == 1) {
                    uint4 v = make_uint4(0, 0, 0, 0);
                    if (there && c * 8 < D) {
                        if (a.aligned) {
                            v = *reinterpret_cast<const uint4 *>(q);
                        } else {
                            R *e = reinterpret_cast<R *>(&v);
#pragma unroll
                            for (int k = 0; k < 8; k++)
                                e[k] = q[k];
                        }
                    }
                    *reinterpret_cast<uint4 *>(to) = v;
                } else {
                    float v[8];
#pragma unroll
                    for (int k = 0; k < 8; k++)
                        v[k] = 0.0f;
                    if (there && c * 8 < D) {
                        if (a.aligned) {
                            *reinterpret_cast<float4 *>(v) = *reinterpret_cast<const float4 *>(q);
                            *reinterpret_cast<float4 *>(v + 4) = *reinterpret_cast<const float4 *>(q + 4);
                        } else {
#pragma unroll
                            for (int k = 0; k < 8; k++)
                                v[k] = to_float(q[k]);
                        }
                    }
                    float unit = a.scale * kTreeLog2e;
                    if constexpr (kHalf) { /* greatest |q| to [2^10, 2^11) */
                        float top = 0.0f;
#pragma unroll
                        for (int k = 0; k < 8; k++)
                            top = fmaxf(top, fabsf(v[k]));
#pragma unroll
                        for (int e = kAcross / 2; e > 0; e >>= 1)
                            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, e));
                        const int e = int(__float_as_uint(top) >> 23);
                        if (e > 0 && e < 255) {
                            const int field = min(264 - e, 253);
                            const float gain = __uint_as_float(uint32_t(field) << 23);
#pragma unroll
                            for (int k = 0; k < 8; k++)
                                v[k] *= gain;
                            unit *= __uint_as_float(uint32_t(254 - field) << 23);
                        }
                    }
                    if (c == 0)
                        sh.unit[r] = unit;
#pragma unroll
                    for (int t = 0; t < kTerms; t++) {
                        uint4 term;
                        uint32_t *e = reinterpret_cast<uint32_t *>(&term);
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            e[k] = Pair<T>::pack(v[2 * k], v[2 * k + 1]);
                            const float2 taken = Pair<T>::unpack(e[k]);
                            v[2 * k] -= taken.x;
                            v[2 * k + 1] -= taken.y;
                        }
                        *reinterpret_cast<uint4 *>(to + t * Plan::kQueryBytes) = term;
                    }
                }
            }
            fence_async();
            mbar_arrive(&sh.queries);
            if constexpr (kTerms > 1)
                everyone(); /* the units */

            const int my_row = both ? w * 128 + row : row; /* of the item */
            const bool counts = my_row < x.rows;
            const bool idle = __all_sync(0xffffffffu, !counts); /* a warp without rows */
            const float unit = kTerms > 1 ? sh.unit[row] : a.scale * kTreeLog2e;
            const uint32_t *seen = a.mask;
            if (counts)
                seen += (int64_t(x.span.row0) + (x.first_row + my_row) / p.group) * a.mask_words;
            /* weights are 2^(logit - from), `from` kLift below a maximum */
            float from = -INFINITY, l = 0.0f;
            const float unseen = unit < 0.0f ? INFINITY : -INFINITY;
            int mine = 0; /* tiles of this stream */
            for (int i = both ? 0 : w; i < n; i += both ? 1 : 2) {
                const uint32_t values = base + place_of_values(i, n);
                const int stage = stage_of(values), t0 = (x.tile0 + i) * kTile;
                if (alive)
                    alive = await(&sh.logits[w], turns & 1) && await(&sh.full[stage], parity_of(values));
                alive = __all_sync(0xffffffffu, alive);
                turns++;
                const bool first = mine++ == 0;
                if (!alive)
                    continue;
                tc_after();
                uint32_t words[kTile / 32];
                bool plain = t0 + kTile <= x.span.prefix;
#pragma unroll
                for (int k = 0; k < kTile / 32; k++) {
                    words[k] = sh.valid[stage][k];
                    plain &= words[k] == ~0u;
                }
                if (!plain && (!both || w == 0)) {
                    /* values that must not meet weights of 0 */
                    const int slot = row;
                    if (slot < kTile) {
                        const bool there = (sh.valid[stage][slot >> 5] >> (slot & 31)) & 1;
                        if (!there || t0 + slot >= x.span.prefix) {
                            bool odd = false;
#pragma unroll
                            for (int c = 0; c < DP / 8; c++) {
                                const uint32_t at = ring_at + stage * Plan::kStage + (c >> 3) * (kTile * 128) + slot * 128 +
                                                    (((c & 7) ^ (slot & 7)) << 4);
                                uint4 v = make_uint4(0, 0, 0, 0);
                                uint32_t *e = reinterpret_cast<uint32_t *>(&v);
                                bool change = !there;
                                if (there) {
                                    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];\n"
                                                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                                                 : "r"(at));
#pragma unroll
                                    for (int k = 0; k < 4; k++) {
                                        constexpr uint32_t kInf = Pair<T>::kInfinite;
                                        if ((e[k] & kInf) == kInf) {
                                            e[k] &= 0xffff0000u;
                                            change = odd = true;
                                        }
                                        if ((e[k] & (kInf << 16)) == kInf << 16) {
                                            e[k] &= 0x0000ffffu;
                                            change = odd = true;
                                        }
                                    }
                                }
                                if (change)
                                    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};\n" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z),
                                                 "r"(v.w)
                                                 : "memory");
                            }
                            if (odd)
                                sh.odd = 1;
                        }
                    }
                    fence_async();
                }
                if (!idle) {
                    float s[kTile];
#pragma unroll
                    for (int k = 0; k < kTile; k += 32)
                        tmem_load32(logits_at + k, s + k);
                    tc_wait_ld();
                    if (!plain)
#pragma unroll
                        for (int k = 0; k < kTile; k += 32) {
                            uint32_t sees = words[k / 32];
                            const int node = t0 + k - x.span.prefix;
                            if (node > -32)
                                sees &= counts ? tree_sees(seen, node, x.span.n) : 0u;
#pragma unroll
                            for (int j = 0; j < 32; j++)
                                s[k + j] = (sees >> j) & 1 ? s[k + j] : unseen;
                        }
                    float top = s[0], other = s[1];
                    if (unit >= 0.0f) {
#pragma unroll
                        for (int k = 2; k < kTile; k += 2) {
                            top = fmaxf(top, s[k]);
                            other = fmaxf(other, s[k + 1]);
                        }
                        top = fmaxf(top, other);
                    } else {
#pragma unroll
                        for (int k = 2; k < kTile; k += 2) {
                            top = fminf(top, s[k]);
                            other = fminf(other, s[k + 1]);
                        }
                        top = fminf(top, other);
                    }
                    /* rounded up, so that beside logits of 2^24 and more no weight passes 2^kLift either */
                    const float to = __fsub_ru(__fmul_ru(top, unit), kLift);
                    const float next = to - from > kSlack || from == -INFINITY ? fmaxf(from, to) : from;
                    if (__any_sync(0xffffffffu, next != from)) {
                        const float keep = from == next ? 1.0f : power2(from - next);
                        l *= keep;
                        from = next;
                        if (!first) /* the products before this tile's logits are complete */
#pragma unroll 1
                            for (int c = 0; c < DP; c += 32) {
                                float o[32];
                                tmem_load32(outputs_at + c, o);
                                tc_wait_ld();
#pragma unroll
                                for (int j = 0; j < 32; j++)
                                    o[j] *= keep;
                                tmem_store32(outputs_at + c, o);
                            }
                    }
                    const float less = from == -INFINITY ? 0.0f : -from;
                    float sum = 0.0f, sum1 = 0.0f;
#pragma unroll
                    for (int k = 0; k < kTile; k += 32) {
                        uint32_t e[kTerms][16];
#pragma unroll
                        for (int j = 0; j < 16; j++) {
                            float w0 = power2(fmaf(s[k + 2 * j], unit, less)), w1 = power2(fmaf(s[k + 2 * j + 1], unit, less));
                            if constexpr (kTerms > 1) {
                                sum += w0;
                                sum1 += w1;
                            }
#pragma unroll
                            for (int t = 0; t < kTerms; t++) {
                                e[t][j] = Pair<T>::pack(w0, w1);
                                const float2 taken = Pair<T>::unpack(e[t][j]);
                                if constexpr (kTerms == 1) {
                                    sum += taken.x;
                                    sum1 += taken.y;
                                } else {
                                    w0 -= taken.x;
                                    w1 -= taken.y;
                                }
                            }
                        }
#pragma unroll
                        for (int t = 0; t < kTerms; t++)
                            tmem_store16(logits_at + t * (kTile / 2) + k / 2, e[t]);
                    }
                    l += sum + sum1;
                    tc_wait_st();
                }
                tc_before();
                mbar_arrive(&sh.weights[w]);
            }
            base += 2 * n;

            /* the end of the item, or of this block's part of it */
            if (mine > 0) {
                if (alive)
                    alive = await(&sh.outputs[w], ends & 1);
                ends++;
            }
            alive = __all_sync(0xffffffffu, alive);
            tc_after();
            sh.maxima[w][row] = from;
            sh.sums[w][row] = l;
            everyone(); /* and all products are done: the queries' place is free */
            const bool odd = sh.odd != 0, whole = x.whole();
            float factor = 1.0f, sum = l, top = from;
            const bool paired = !both && n > 1;
            if (paired) {
                const float m1 = sh.maxima[1 - w][row], l1 = sh.sums[1 - w][row];
                top = fmaxf(from, m1);
                const float least = top == -INFINITY ? 0.0f : top;
                const float f = exp2f(from - least), f1 = exp2f(m1 - least);
                /* in the same order in both streams */
                sum = w == 0 ? fmaf(l, f, l1 * f1) : fmaf(l1, f1, l * f);
                factor = f;
            }
            if (whole)
                factor *= sum == 0.0f ? 0.0f : 1.0f / sum;
            if (paired) {
                /* each stream hands the other the half of the dims that it does not finish */
                if (!idle && alive) {
#pragma unroll 1
                    for (int c = 0; c < DP / 2; c += 32) {
                        const int d0 = (w == 0 ? DP / 2 : 0) + c;
                        float o[32];
                        tmem_load32(outputs_at + d0, o);
                        tc_wait_ld();
#pragma unroll
                        for (int j = 0; j < 32; j += 4) {
                            const int piece = (d0 + j) / 4;
                            float4 v = make_float4(o[j] * factor, o[j + 1] * factor, o[j + 2] * factor, o[j + 3] * factor);
                            if (factor == 0.0f)
                                v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                            *reinterpret_cast<float4 *>(smem + row * DP * 4 + ((piece ^ (row & 7)) << 4)) = v;
                        }
                    }
                }
                everyone();
            }
            if (!idle && alive && (both || paired || w == 0)) {
                const TreePart part = tree_part(a, blockIdx.x, x.first <= start ? 0 : 1, x.rows);
                int64_t out_row = 0;
                int h = 0;
                if (counts)
                    tree_row(a, x.span.row0, x.head, x.first_row + my_row, out_row, h);
                if (counts && (both || w == 0)) {
                    if (whole) {
                        if (a.lse)
                            a.lse[out_row * p.heads + h] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * kTreeLn2;
                    } else {
                        part.maxima[my_row] = top;
                        part.sums[my_row] = sum;
                    }
                }
                const int d_from = paired && w == 1 ? DP / 2 : 0, d_to = paired && w == 0 ? DP / 2 : DP;
#pragma unroll 1
                for (int d0 = d_from; d0 < d_to; d0 += 32) {
                    float o[32];
                    tmem_load32(outputs_at + d0, o);
                    tc_wait_ld();
#pragma unroll
                    for (int j = 0; j < 32; j += 4) {
                        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        if (paired)
                            v = *reinterpret_cast<const float4 *>(smem + row * DP * 4 + ((((d0 + j) / 4) ^ (row & 7)) << 4));
                        if (factor != 0.0f)
                            v = make_float4(fmaf(o[j], factor, v.x), fmaf(o[j + 1], factor, v.y), fmaf(o[j + 2], factor, v.z),
                                            fmaf(o[j + 3], factor, v.w));
                        o[j] = v.x;
                        o[j + 1] = v.y;
                        o[j + 2] = v.z;
                        o[j + 3] = v.w;
                    }
                    if (odd && counts) {
                        /* infinities and NaN among the drafted tokens that the row sees */
                        for (int t = max(x.span.prefix, x.tile0 * kTile); t < min(x.span.length, x.tile1 * kTile); t++) {
                            const int node = t - x.span.prefix, page = lookup(p, x.sequence, t / p.page_size);
                            if (page < 0 || !((seen[node >> 5] >> (node & 31)) & 1))
                                continue;
                            const T *v = static_cast<const T *>(p.values) + int64_t(page) * p.page_stride +
                                         int64_t(x.head) * p.head_stride + int64_t(t % p.page_size) * p.slot_stride;
#pragma unroll
                            for (int j = 0; j < 32; j++)
                                if (d0 + j < D) {
                                    const float e = to_float(v[d0 + j]);
                                    o[j] += fabsf(e) <= 3.402823466e38f ? 0.0f : e;
                                }
                        }
                    }
                    if (!counts)
                        continue;
                    if (!whole) {
                        float *to = part.out + int64_t(my_row) * D + d0;
#pragma unroll
                        for (int j = 0; j < 32; j += 4)
                            if (d0 + j < D)
                                *reinterpret_cast<float4 *>(to + j) = make_float4(o[j], o[j + 1], o[j + 2], o[j + 3]);
                    } else {
                        R *to = static_cast<R *>(a.out) + out_row * a.out_stride + int64_t(h) * D + d0;
                        constexpr int kPer = 16 / sizeof(R);
#pragma unroll
                        for (int j = 0; j < 32; j += kPer)
                            if (d0 + j < D) {
                                uint4 v;
                                R *e = reinterpret_cast<R *>(&v);
#pragma unroll
                                for (int k = 0; k < kPer; k++)
                                    e[k] = output_of<R>(o[j + k]);
                                if (a.aligned) {
                                    *reinterpret_cast<uint4 *>(to + j) = v;
                                } else {
#pragma unroll
                                    for (int k = 0; k < kPer; k++)
                                        to[j + k] = e[k];
                                }
                            }
                    }
                }
            }
            if (!whole && x.tile0 == 0)
                join = tree_join(x, share);
            everyone(); /* the statistics and the queries' place are free again */
            if (tid == 0)
                sh.odd = 0;
            tc_before();
        }
        if (tid == 0)
            a.joins[blockIdx.x] = join;
    }
    tc_before();
    __syncthreads();
    if (warp == kIssuer) {
        tc_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;\n" ::"r"(tmem) : "memory");
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
    e = launch_kernel(kernel, dim3(a.sms), kThreads, Plan::kBytes, s, 1, a);
    return e != cudaSuccess ? e : tree_join_parts(a, a.sms, Plan::kBlockRows, s);
}

} // namespace

cudaError_t paged_tree_tc(const PagedTree &a, cudaStream_t s) {
    const bool narrow = a.p.head_dim <= 64;
    if (a.p.type == 1) {
        if (a.type == 0)
            return narrow ? launch<__half, float, 64, 2>(a, s) : launch<__half, float, 128, 2>(a, s);
        return narrow ? launch<__half, __half, 64, 1>(a, s) : launch<__half, __half, 128, 1>(a, s);
    }
    if (a.type == 0)
        return narrow ? launch<__nv_bfloat16, float, 64, 3>(a, s) : launch<__nv_bfloat16, float, 128, 3>(a, s);
    return narrow ? launch<__nv_bfloat16, __nv_bfloat16, 64, 1>(a, s) : launch<__nv_bfloat16, __nv_bfloat16, 128, 1>(a, s);
}

} // namespace nut
