/* C ABI of the paged KV cache (nut_paged_* in nutllm_cuda.h): argument
 * checks, the handle's workspace, and the calls into paged_*.cu. */
#include <algorithm>
#include <climits>
#include <cmath>
#include <memory>
#include <mutex>
#include <stdexcept>
#include <string>

#include <cuda_runtime.h>

#include "../../include/nutllm_cuda.h"
#include "kernels.h"
#include "paged.h"

namespace {

struct Failure {
    nut_status status;
    std::string message;
};

[[noreturn]] void raise(nut_status s, const std::string &m) { throw Failure{s, "paged: " + m}; }

void cuda_check(cudaError_t e, const char *what) {
    if (e != cudaSuccess) {
        cudaGetLastError(); /* reported here: the next call's own check is not to find it */
        throw Failure{NUT_RUNTIME_ERROR,
                      std::string("cuda: ") + what + ": " + cudaGetErrorString(e)};
    }
}

template <typename F> nut_status guarded(F &&body) {
    try {
        body();
        return NUT_OK;
    } catch (const Failure &f) {
        nut::set_last_error(f.message);
        return f.status;
    } catch (const std::bad_alloc &) {
        nut::set_last_error("nutllm: host allocation failed");
        return NUT_RUNTIME_ERROR;
    } catch (const std::exception &e) {
        nut::set_last_error(e.what());
        return NUT_RUNTIME_ERROR;
    }
}

/* Makes the handle's device current where it is not, and restores it. */
struct DeviceScope {
    int previous = 0, device;
    explicit DeviceScope(int d) : device(d) {
        cuda_check(cudaGetDevice(&previous), "get device");
        if (previous != device)
            cuda_check(cudaSetDevice(device), "set device");
    }
    ~DeviceScope() {
        if (previous != device)
            cudaSetDevice(previous);
    }
};

/* Workspaces come from a memory pool of this library's own on each device,
 * which keeps up to 64 MB that handles gave back: a handle is made in some 20
 * us, where cudaMalloc and cudaFree take 300 to 400 each. */
cudaMemPool_t workspace_pool(int device) {
    static std::mutex lock;
    static cudaMemPool_t pools[nut::kMaxDevices] = {};
    if (device < 0 || device >= nut::kMaxDevices)
        raise(NUT_INVALID_ARGUMENT, "device out of range");
    const std::lock_guard<std::mutex> hold(lock);
    if (!pools[device]) {
        cudaMemPoolProps props{};
        props.allocType = cudaMemAllocationTypePinned;
        props.location.type = cudaMemLocationTypeDevice;
        props.location.id = device;
        cuda_check(cudaMemPoolCreate(&pools[device], &props), "create workspace pool");
        uint64_t keep = uint64_t(64) << 20;
        cuda_check(cudaMemPoolSetAttribute(pools[device], cudaMemPoolAttrReleaseThreshold, &keep),
                   "size workspace pool");
    }
    return pools[device];
}

constexpr int64_t kMaxGrid = 65535; /* sequences and rows are grid dimensions */

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

void check_view(const nut_paged_view &v) {
    if (!v.keys || !v.values || !v.table || !v.lengths)
        raise(NUT_INVALID_ARGUMENT, "null pool, table or lengths");
    if ((v.bounds == nullptr) != (v.bound_scales == nullptr))
        raise(NUT_INVALID_ARGUMENT, "bounds and bound_scales go together");
    if (v.type != NUT_F32 && v.type != NUT_F16 && v.type != NUT_BF16)
        raise(NUT_INVALID_ARGUMENT, "unknown cache type");
    if (v.sequences <= 0 || v.max_pages <= 0 || v.n_pages <= 0 || v.page_size <= 0 ||
        v.heads <= 0 || v.kv_heads <= 0 || v.head_dim <= 0 || v.max_rows < 0)
        raise(NUT_INVALID_ARGUMENT, "invalid dimensions");
    if (v.heads % v.kv_heads != 0)
        raise(NUT_INVALID_ARGUMENT, "heads must divide by kv_heads");
    if (v.head_dim % 8 != 0 || v.head_dim > 256)
        raise(NUT_INVALID_ARGUMENT, "head_dim must be a multiple of 8 up to 256");
    if (v.sequences > kMaxGrid || v.max_rows > kMaxGrid || v.kv_heads > 4096 || v.heads > 65536)
        raise(NUT_LENGTH_ERROR, "dimensions exceed device limits");
    /* strides of 2^36 elements stay within a tensor map's 2^40 bytes */
    if (std::max({v.page_stride, v.head_stride, v.slot_stride}) >= (int64_t(1) << 36) ||
        v.kv_heads * v.page_size * v.head_dim >= (int64_t(1) << 36))
        raise(NUT_LENGTH_ERROR, "strides exceed device limits");
    if (v.n_pages > INT_MAX || v.page_size > (1 << 24) || v.max_pages > (1 << 24) ||
        v.max_pages * v.page_size > (int64_t(1) << 30))
        raise(NUT_LENGTH_ERROR, "dimensions exceed device limits");
    const int64_t unit = v.type == NUT_F32 ? 4 : 8; /* elements of 16 bytes */
    if (!aligned16(v.keys) || !aligned16(v.values) || v.page_stride % unit != 0 ||
        v.head_stride % unit != 0 || v.slot_stride % unit != 0)
        raise(NUT_INVALID_ARGUMENT, "keys, values and strides must be multiples of 16 bytes");
    if (!aligned16(v.bounds))
        raise(NUT_INVALID_ARGUMENT, "bounds must be a multiple of 16 bytes");
    if (v.page_stride < 0 || v.head_stride < 0 || v.slot_stride < 0)
        raise(NUT_INVALID_ARGUMENT, "negative stride");
    if ((v.page_stride || v.head_stride || v.slot_stride) &&
        !(v.page_stride && v.head_stride && v.slot_stride))
        raise(NUT_INVALID_ARGUMENT, "give all three strides or none");
}

/* cuTensorMapEncodeTiled through the runtime: the library does not link the
 * driver library. */
using EncodeTiled = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                 const cuuint64_t *, const cuuint32_t *, const cuuint32_t *,
                                 CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                                 CUtensorMapFloatOOBfill);

/* The pool as the attention's tensor map (PagedAttention::key_map); dims
 * behind head_dim read as zeros. */
CUtensorMap pool_map(const nut::PagedPool &p, void *base, int box, bool whole) {
    static const EncodeTiled encode = [] {
        void *f = nullptr;
        cudaDriverEntryPointQueryResult q{};
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            f = nullptr;
        return reinterpret_cast<EncodeTiled>(f);
    }();
    if (!encode)
        raise(NUT_RUNTIME_ERROR, "the driver has no cuTensorMapEncodeTiled");
    const cuuint64_t size = p.type == NUT_F32 ? 4 : 2;
    const CUtensorMapDataType type = p.type == NUT_F32   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                     : p.type == NUT_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                         : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    const int width = int(128 / size);
    const cuuint64_t dims[5] = {cuuint64_t(whole ? width : p.head_dim), cuuint64_t(p.page_size),
                                cuuint64_t(whole ? p.head_dim / width : 1), cuuint64_t(p.kv_heads),
                                cuuint64_t(p.n_pages)};
    const cuuint64_t strides[4] = {cuuint64_t(p.slot_stride) * size, 128, cuuint64_t(p.head_stride) * size,
                                   cuuint64_t(p.page_stride) * size};
    const cuuint32_t columns = cuuint32_t(nut::paged_columns(p.type, p.head_dim));
    const cuuint32_t boxes[5] = {cuuint32_t(width), cuuint32_t(box), whole ? columns : 1, 1, 1};
    const cuuint32_t steps[5] = {1, 1, 1, 1, 1};
    CUtensorMap map;
    if (encode(&map, type, 5, base, dims, strides, boxes, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        raise(NUT_INVALID_ARGUMENT, "the pool's strides cannot be mapped");
    return map;
}

/* Row stride in elements: 0 stands for the contiguous width. */
int64_t stride_of(int64_t given, int64_t width, const char *name) {
    if (given == 0)
        return width;
    if (given < width)
        raise(NUT_INVALID_ARGUMENT, std::string(name) + " is less than a row");
    return given;
}

} // namespace

struct nut_paged {
    int device = 0;
    nut::PagedPool pool{};
    CUtensorMap key_map{}, value_map{};
    int box = 16;
    bool whole_columns = false;
    uint64_t page_magic = 0;
    int page_shift = 32;
    int max_rows = 0;
    bool track = false;
    int sms = 0;
    char *block = nullptr; /* one allocation, cut into the parts below */
    int *error = nullptr, *counters = nullptr;
    float *partial = nullptr, *logits = nullptr, *lse2 = nullptr, *scores = nullptr;
    int32_t *pairs = nullptr, *counts = nullptr;
    ~nut_paged() {
        if (block) {
            cudaDeviceSynchronize(); /* calls in flight, on any stream, still use it */
            cudaFreeAsync(block, nullptr);
        }
    }
};

namespace {

void check_row_type(const nut_paged &h, int32_t type) {
    if (type != NUT_F32 && type != h.pool.type)
        raise(NUT_INVALID_ARGUMENT, "rows must be fp32 or of the cache's type");
}

void check_rows(const nut_paged &h, int64_t rows, const int32_t *row_sequence) {
    if (rows < 0)
        raise(NUT_INVALID_ARGUMENT, "negative row count");
    if (rows > h.max_rows)
        raise(NUT_LENGTH_ERROR, "more rows than max_rows");
    if (!row_sequence && rows > h.pool.sequences)
        raise(NUT_INVALID_ARGUMENT, "more rows than sequences need row_sequence");
}

} // namespace

extern "C" {

nut_status nut_paged_create(const nut_paged_view *view, int device, nut_paged **out) {
    return guarded([&] {
        if (!view || !out)
            raise(NUT_INVALID_ARGUMENT, "null argument");
        *out = nullptr;
        check_view(*view);
        const nut_paged_view &v = *view;
        DeviceScope scope(device);
        auto h = std::make_unique<nut_paged>();
        h->device = device;
        h->max_rows = int(v.max_rows ? v.max_rows : v.sequences);
        h->track = v.track_weights != 0;
        nut::PagedPool &p = h->pool;
        p.keys = v.keys;
        p.values = v.values;
        p.table = v.table;
        p.lengths = v.lengths;
        p.bounds = v.bounds;
        p.bound_scales = v.bound_scales;
        const bool strided = v.page_stride != 0;
        p.slot_stride = strided ? v.slot_stride : v.head_dim;
        p.head_stride = strided ? v.head_stride : v.page_size * v.head_dim;
        p.page_stride = strided ? v.page_stride : v.kv_heads * v.page_size * v.head_dim;
        p.sequences = int(v.sequences);
        p.max_pages = int(v.max_pages);
        p.n_pages = int(v.n_pages);
        p.page_size = int(v.page_size);
        p.heads = int(v.heads);
        p.kv_heads = int(v.kv_heads);
        p.head_dim = int(v.head_dim);
        p.group = int(v.heads / v.kv_heads);
        p.capacity = int(v.max_pages * v.page_size);
        p.type = v.type;
        cuda_check(cudaDeviceGetAttribute(&h->sms, cudaDevAttrMultiProcessorCount, device),
                   "count SMs");
        h->sms = std::min(h->sms, nut::kMaxSms);
        while (p.page_size % h->box != 0)
            h->box /= 2;
        /* ceil(2^(32 + s) / page_size) with 2^s < page_size <= 2^(s + 1): exact below 2^31 */
        while ((int64_t(1) << (h->page_shift - 31)) < p.page_size)
            h->page_shift++;
        h->page_magic = ((uint64_t(1) << h->page_shift) + p.page_size - 1) / p.page_size;
        h->whole_columns = h->box == 16 && p.head_dim % (p.type == NUT_F32 ? 32 : 64) == 0;
        h->key_map = pool_map(p, p.keys, h->box, h->whole_columns);
        h->value_map = pool_map(p, p.values, h->box, h->whole_columns);
        const size_t items = size_t(p.sequences) * p.kv_heads;
        size_t bytes = 0;
        const auto part = [&](size_t count, size_t size) {
            const size_t at = bytes;
            bytes += (count * size + 255) / 256 * 256;
            return at;
        };
        /* zeroed at first: the error word and the counters */
        const size_t error = part(1, 4);
        const size_t counters = part(size_t(h->max_rows) * p.kv_heads * ((p.group + 7) / 8), 4);
        const size_t zeroed = bytes;
        const size_t partial = part(size_t(h->sms) * nut::kMaxCtasPerSm * 2 *
                                        nut::paged_part_floats(nut::paged_padded_dim(p.type, p.head_dim)),
                                    4);
        const size_t pairs = part(items * p.capacity, 4), counts = part(items * 2, 4);
        const size_t logits = part(h->track ? size_t(p.sequences) * p.heads * p.capacity : 0, 4);
        const size_t lse2 = part(h->track ? size_t(p.sequences) * p.heads : 0, 4);
        const size_t scores = part(p.bounds ? size_t(h->max_rows) * p.kv_heads * p.max_pages : 0, 4);
        void *block = nullptr;
        cuda_check(cudaMallocFromPoolAsync(&block, bytes, workspace_pool(device), nullptr), "alloc workspace");
        h->block = static_cast<char *>(block);
        const auto floats = [&](size_t at) { return reinterpret_cast<float *>(h->block + at); };
        const auto ints = [&](size_t at) { return reinterpret_cast<int32_t *>(h->block + at); };
        p.error = h->error = ints(error);
        h->counters = ints(counters);
        h->partial = floats(partial);
        h->pairs = ints(pairs);
        h->counts = ints(counts);
        h->logits = floats(logits);
        h->lse2 = floats(lse2);
        h->scores = floats(scores);
        cuda_check(cudaMemsetAsync(h->block, 0, zeroed, nullptr), "clear workspace");
        cuda_check(cudaStreamSynchronize(nullptr), "finish workspace");
        *out = h.release();
    });
}

nut_status nut_paged_destroy(nut_paged *h) {
    return guarded([&] {
        if (!h)
            return;
        DeviceScope scope(h->device);
        delete h;
    });
}

nut_status nut_paged_error(nut_paged *h, void *stream) {
    return guarded([&] {
        if (!h)
            raise(NUT_INVALID_ARGUMENT, "null handle");
        DeviceScope scope(h->device);
        const cudaStream_t s = static_cast<cudaStream_t>(stream);
        int code = 0;
        cuda_check(cudaMemcpyAsync(&code, h->error, sizeof code, cudaMemcpyDeviceToHost, s),
                   "read error word");
        cuda_check(cudaStreamSynchronize(s), "synchronize");
        if (code == 0)
            return;
        cuda_check(cudaMemsetAsync(h->error, 0, sizeof code, s), "clear error word");
        cuda_check(cudaStreamSynchronize(s), "synchronize");
        if (code & nut::kPagedTimeout)
            raise(NUT_DEVICE_TIMEOUT, "a copy from the pool did not arrive");
        std::string m;
        const auto add = [&](int bit, const char *what) {
            if (code & bit)
                m += (m.empty() ? "" : ", ") + std::string(what);
        };
        add(nut::kPagedBadPage, "page number outside the pool");
        add(nut::kPagedBadLength, "length outside the table");
        add(nut::kPagedBadSequence, "row sequence out of range");
        add(nut::kPagedBadStarts, "inconsistent starts");
        add(nut::kPagedBadPosition, "position outside the rotation table");
        raise(NUT_OUT_OF_RANGE, m);
    });
}

nut_status nut_paged_append(nut_paged *h, const nut_paged_append_args *args, void *stream) {
    return guarded([&] {
        if (!h || !args)
            raise(NUT_INVALID_ARGUMENT, "null argument");
        const nut_paged_append_args &g = *args;
        const nut::PagedPool &p = h->pool;
        if (!g.k || !g.v || !g.starts)
            raise(NUT_INVALID_ARGUMENT, "null keys, values or starts");
        if ((g.q == nullptr) != (g.q_out == nullptr))
            raise(NUT_INVALID_ARGUMENT, "q and q_out go together");
        if ((g.rope_cos == nullptr) != (g.rope_sin == nullptr))
            raise(NUT_INVALID_ARGUMENT, "rope_cos and rope_sin go together");
        if (g.rope_cos && g.rope_rows <= 0)
            raise(NUT_INVALID_ARGUMENT, "empty rotation table");
        if (g.rows < 0 || g.max_new < 0)
            raise(NUT_INVALID_ARGUMENT, "negative row count");
        check_row_type(*h, g.type);
        nut::PagedAppend a{};
        a.p = p;
        const int64_t D = p.head_dim;
        a.q_stride = stride_of(g.q_stride, p.heads * D, "q_stride");
        a.k_stride = stride_of(g.k_stride, p.kv_heads * D, "k_stride");
        a.v_stride = stride_of(g.v_stride, p.kv_heads * D, "v_stride");
        a.q_out_stride = stride_of(g.q_out_stride, p.heads * D, "q_out_stride");
        if (g.rows > INT_MAX)
            raise(NUT_LENGTH_ERROR, "too many rows");
        if (g.max_new > p.capacity)
            raise(NUT_LENGTH_ERROR, "more new tokens than a sequence can hold");
        /* a block counts a page's rows and steps beyond them by its threads */
        if (std::min<int64_t>(g.max_new, p.page_size) * ((g.q ? p.group : 0) + 2) > INT_MAX - 1024)
            raise(NUT_LENGTH_ERROR, "too many rows for one page: append fewer at a time");
        if (g.rows == 0 || g.max_new == 0)
            return;
        a.q = g.q;
        a.k = g.k;
        a.v = g.v;
        a.q_out = g.q_out;
        a.starts = g.starts;
        a.seen = g.seen;
        a.cos = g.rope_cos;
        a.sin = g.rope_sin;
        a.rows = int(g.rows);
        a.max_new = int(g.max_new);
        a.rope_rows = int(std::min<int64_t>(g.rope_rows, INT_MAX));
        a.type = g.type;
        a.positions = g.positions;
        a.weights = g.weights;
        DeviceScope scope(h->device);
        cuda_check(nut::paged_append(a, static_cast<cudaStream_t>(stream)), "paged append");
    });
}

nut_status nut_paged_summarise(nut_paged *h, void *stream) {
    return guarded([&] {
        if (!h)
            raise(NUT_INVALID_ARGUMENT, "null handle");
        if (!h->pool.bounds)
            raise(NUT_INVALID_ARGUMENT, "the pool has no bounds");
        DeviceScope scope(h->device);
        cuda_check(nut::paged_summarise(h->pool, static_cast<cudaStream_t>(stream)),
                   "paged summarise");
    });
}

nut_status nut_paged_attention(nut_paged *h, const nut_paged_attention_args *args, void *stream) {
    return guarded([&] {
        if (!h || !args)
            raise(NUT_INVALID_ARGUMENT, "null argument");
        const nut_paged_attention_args &g = *args;
        const nut::PagedPool &p = h->pool;
        if (!g.q || !g.out)
            raise(NUT_INVALID_ARGUMENT, "null q or out");
        check_row_type(*h, g.type);
        check_rows(*h, g.rows, g.row_sequence);
        if (g.selected && g.n_selected <= 0)
            raise(NUT_INVALID_ARGUMENT, "n_selected must be positive");
        if (g.selected && g.n_selected > (int64_t(1) << 30) / p.page_size)
            raise(NUT_LENGTH_ERROR, "too many selected pages");
        /* the kernel counts tiles of at least 32 slots, and 3 for each item, in 32 bits; its
         * blocks' shares are rounded up, and pass the end by less than a place a block */
        const int64_t slots = g.selected ? g.n_selected * p.page_size : p.capacity;
        if (g.rows * p.kv_heads * ((p.group + 7) / 8) * (slots / 32 + 4) >
            INT_MAX - nut::kMaxSms * nut::kMaxCtasPerSm)
            raise(NUT_LENGTH_ERROR, "too many rows for so long a table: split the call");
        if ((g.weights == nullptr) != (g.weights_out == nullptr))
            raise(NUT_INVALID_ARGUMENT, "weights and weights_out go together");
        if (g.weights && !h->track)
            raise(NUT_INVALID_ARGUMENT, "the handle does not track weights");
        if (g.weights && (g.selected || g.row_sequence))
            raise(NUT_INVALID_ARGUMENT, "weights need one row per sequence over all of its pages");
        if (!std::isfinite(g.scale))
            raise(NUT_INVALID_ARGUMENT, "scale must be finite");
        nut::PagedAttention a{};
        a.p = p;
        a.q_stride = stride_of(g.q_stride, int64_t(p.heads) * p.head_dim, "q_stride");
        a.out_stride = stride_of(g.out_stride, int64_t(p.heads) * p.head_dim, "out_stride");
        if (g.rows == 0)
            return;
        a.q = g.q;
        a.out = g.out;
        a.lse = g.lse;
        a.row_sequence = g.row_sequence;
        a.row_length = g.row_length;
        a.selected = g.selected;
        a.n_selected = g.selected ? int(g.n_selected) : 0;
        a.weights = g.weights;
        a.weights_out = g.weights_out;
        a.rows = int(g.rows);
        a.type = g.type;
        a.scale = g.scale != 0.0f ? g.scale : float(1.0 / std::sqrt(double(p.head_dim)));
        a.logits = h->logits;
        a.lse2 = h->lse2;
        a.partial = h->partial;
        a.counters = h->counters;
        a.sms = h->sms;
        a.key_map = h->key_map;
        a.value_map = h->value_map;
        a.box = h->box;
        a.whole_columns = h->whole_columns;
        a.page_shift = h->page_shift;
        a.page_magic = h->page_magic;
        DeviceScope scope(h->device);
        cuda_check(nut::paged_attention(a, static_cast<cudaStream_t>(stream)), "paged attention");
    });
}

nut_status nut_paged_select(nut_paged *h, const nut_paged_select_args *args, void *stream) {
    return guarded([&] {
        if (!h || !args)
            raise(NUT_INVALID_ARGUMENT, "null argument");
        const nut_paged_select_args &g = *args;
        const nut::PagedPool &p = h->pool;
        if (!p.bounds)
            raise(NUT_INVALID_ARGUMENT, "the pool has no bounds");
        if (!g.q || !g.selected)
            raise(NUT_INVALID_ARGUMENT, "null q or selected");
        check_row_type(*h, g.type);
        check_rows(*h, g.rows, g.row_sequence);
        if (g.n_selected <= 0 || g.sink_pages < 0 || g.recent_pages < 0)
            raise(NUT_INVALID_ARGUMENT, "invalid page counts");
        if (g.n_selected > INT_MAX)
            raise(NUT_LENGTH_ERROR, "too many selected pages");
        nut::PagedSelect a{};
        a.p = p;
        a.q_stride = stride_of(g.q_stride, int64_t(p.heads) * p.head_dim, "q_stride");
        if (g.rows == 0)
            return;
        a.q = g.q;
        a.row_sequence = g.row_sequence;
        a.row_length = g.row_length;
        a.selected = g.selected;
        a.n_selected = int(g.n_selected);
        a.sink_pages = int(std::min<int64_t>(g.sink_pages, INT_MAX));
        a.recent_pages = int(std::min<int64_t>(g.recent_pages, INT_MAX));
        a.rows = int(g.rows);
        a.type = g.type;
        a.scores = h->scores;
        DeviceScope scope(h->device);
        cuda_check(nut::paged_select(a, static_cast<cudaStream_t>(stream)), "paged select");
    });
}

nut_status nut_paged_evict(nut_paged *h, const nut_paged_evict_args *args, void *stream) {
    return guarded([&] {
        if (!h || !args)
            raise(NUT_INVALID_ARGUMENT, "null argument");
        const nut_paged_evict_args &g = *args;
        if (!g.weights || !g.weights_out || !g.new_lengths)
            raise(NUT_INVALID_ARGUMENT, "null weights, weights_out or new_lengths");
        if ((g.positions == nullptr) != (g.positions_out == nullptr))
            raise(NUT_INVALID_ARGUMENT, "positions and positions_out go together");
        if (g.budget < 0 || g.sinks < 0 || g.recent < 0)
            raise(NUT_INVALID_ARGUMENT, "negative budget, sinks or recent");
        if ((g.sinks || g.recent) && !g.positions)
            raise(NUT_INVALID_ARGUMENT, "sinks and recent need positions");
        if (g.recent && !g.seen)
            raise(NUT_INVALID_ARGUMENT, "recent needs seen");
        nut::PagedEvict a{};
        a.p = h->pool;
        a.weights = g.weights;
        a.positions = g.positions;
        a.seen = g.seen;
        a.budget = int(std::min<int64_t>(g.budget, INT_MAX));
        a.sinks = int(std::min<int64_t>(g.sinks, INT_MAX));
        a.recent = int(std::min<int64_t>(g.recent, INT_MAX));
        a.new_lengths = g.new_lengths;
        a.weights_out = g.weights_out;
        a.positions_out = g.positions_out;
        a.pairs = h->pairs;
        a.counts = h->counts;
        DeviceScope scope(h->device);
        cuda_check(nut::paged_evict(a, static_cast<cudaStream_t>(stream)), "paged evict");
    });
}

} // extern "C"
