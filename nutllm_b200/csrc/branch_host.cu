/* C ABI of branching sequences' pages (nut_pages_*) and of beam selection
 * (nut_beam_*): argument checks, workspaces, and the calls into pages.cu and
 * beam.cu. */
#include <algorithm>
#include <climits>
#include <memory>
#include <string>

#include <cuda_runtime.h>

#include "abi.h"
#include "branch.h"

using namespace nut::abi;

/* One allocation, cut into parts. */
struct Workspace {
    char *block = nullptr;
    size_t bytes = 0;
    size_t part(size_t count, size_t size) {
        const size_t at = bytes;
        bytes += (count * size + 255) / 256 * 256;
        return at;
    }
    void make(int device, size_t zeroed) {
        void *p = nullptr;
        cuda_check(cudaMallocFromPoolAsync(&p, bytes, workspace_pool(device), nullptr), "alloc workspace");
        block = static_cast<char *>(p);
        cuda_check(cudaMemsetAsync(block, 0, zeroed, nullptr), "clear workspace");
        cuda_check(cudaStreamSynchronize(nullptr), "finish workspace");
    }
    ~Workspace() {
        if (block) {
            cudaDeviceSynchronize(); /* calls in flight, on any stream, still use it */
            cudaFreeAsync(block, nullptr);
        }
    }
};

struct nut_pages {
    int device = 0;
    nut::PagesUpdate u{};
    Workspace space;
};

struct nut_beam {
    int device = 0;
    nut::BeamSelect b{};
    Workspace space;
};

namespace {

constexpr int64_t kMostRows = 65535; /* a grid dimension */

[[noreturn]] void refuse(nut_status s, const char *what, const std::string &m) {
    throw Failure{s, std::string(what) + ": " + m};
}

} // namespace

extern "C" {

nut_status nut_pages_create(const nut_pages_view *view, int device, nut_pages **out) {
    return guarded([&] {
        if (!view || !out)
            refuse(NUT_INVALID_ARGUMENT, "pages", "null argument");
        *out = nullptr;
        const nut_pages_view &v = *view;
        if (!v.table || !v.lengths || !v.refs || !v.free_pages || !v.free_count)
            refuse(NUT_INVALID_ARGUMENT, "pages", "null table, lengths, refs, free_pages or free_count");
        if (!aligned4({v.table, v.lengths, v.refs, v.free_pages, v.free_count}))
            refuse(NUT_INVALID_ARGUMENT, "pages", "arrays must be multiples of their elements");
        if (v.sequences <= 0 || v.max_pages <= 0 || v.n_pages <= 0 || v.page_size <= 0)
            refuse(NUT_INVALID_ARGUMENT, "pages", "invalid dimensions");
        if (v.sequences > kMostRows || v.n_pages > INT_MAX - 4096 || v.page_size > (1 << 24) ||
            v.max_pages > (1 << 24) || v.max_pages * v.page_size > (int64_t(1) << 30))
            refuse(NUT_LENGTH_ERROR, "pages", "dimensions exceed device limits");
        DeviceScope scope(device);
        auto h = std::make_unique<nut_pages>();
        h->device = device;
        nut::PagesUpdate &u = h->u;
        u.table = v.table;
        u.lengths = v.lengths;
        u.refs = v.refs;
        u.free_pages = v.free_pages;
        u.free_count = v.free_count;
        u.sequences = int(v.sequences);
        u.max_pages = int(v.max_pages);
        u.n_pages = int(v.n_pages);
        u.page_size = int(v.page_size);
        Workspace &w = h->space;
        const size_t pages = size_t(v.n_pages), sequences = size_t(v.sequences);
        const size_t words = w.part(2, 4), delta = w.part(pages, 4), writers = w.part(pages, 4),
                     first = w.part(pages, 4);
        const size_t zeroed = w.bytes;
        const size_t plan = w.part(sequences, sizeof(int4)), freed = w.part(nut::kPagesMostWarps, 4),
                     staged = w.part(sequences * size_t(v.max_pages), 4), changes = w.part(sequences, 4);
        w.make(device, zeroed);
        const auto ints = [&](size_t at) { return reinterpret_cast<int32_t *>(w.block + at); };
        u.met = ints(words);
        u.error = u.met + 1;
        u.delta = ints(delta);
        u.writers = ints(writers);
        u.first = ints(first);
        u.plan = reinterpret_cast<int4 *>(w.block + plan);
        u.freed = ints(freed);
        u.staged = ints(staged);
        u.changes = ints(changes);
        *out = h.release();
    });
}

nut_status nut_pages_destroy(nut_pages *h) {
    return guarded([&] {
        if (!h)
            return;
        DeviceScope scope(h->device);
        delete h;
    });
}

nut_status nut_pages_error(nut_pages *h, void *stream) {
    return guarded([&] {
        if (!h)
            refuse(NUT_INVALID_ARGUMENT, "pages", "null handle");
        DeviceScope scope(h->device);
        const cudaStream_t s = static_cast<cudaStream_t>(stream);
        int code = 0;
        cuda_check(cudaMemcpyAsync(&code, h->u.error, sizeof code, cudaMemcpyDeviceToHost, s), "read error word");
        cuda_check(cudaStreamSynchronize(s), "synchronize");
        if (code == 0)
            return;
        cuda_check(cudaMemsetAsync(h->u.error, 0, sizeof code, s), "clear error word");
        cuda_check(cudaStreamSynchronize(s), "synchronize");
        std::string m;
        const auto add = [&](int bit, const char *what) {
            if (code & bit)
                m += (m.empty() ? "" : ", ") + std::string(what);
        };
        add(nut::kPagesBadArgument, "parent, keep or add out of range");
        add(nut::kPagesBadLength, "length outside the table");
        add(nut::kPagesBadPage, "page number, holders or free pages out of range");
        add(nut::kPagesNoneFree, "not enough free pages");
        refuse(code == nut::kPagesNoneFree ? NUT_LENGTH_ERROR : NUT_OUT_OF_RANGE, "pages", m);
    });
}

nut_status nut_pages_update(nut_pages *h, const nut_pages_update_args *args, void *stream) {
    return guarded([&] {
        if (!h || !args)
            refuse(NUT_INVALID_ARGUMENT, "pages", "null argument");
        const nut_pages_update_args &g = *args;
        const bool lists = g.copy_from && g.copy_to && g.copy_slots;
        if (!lists && (g.copy_from || g.copy_to || g.copy_slots))
            refuse(NUT_INVALID_ARGUMENT, "pages", "copy_from, copy_to and copy_slots go together");
        if (!lists && g.add)
            refuse(NUT_INVALID_ARGUMENT, "pages", "add needs the copy lists");
        if (!aligned4({g.parent, g.keep, g.add, g.copy_from, g.copy_to, g.copy_slots}))
            refuse(NUT_INVALID_ARGUMENT, "pages", "arrays must be multiples of their elements");
        nut::PagesUpdate u = h->u;
        u.parent = g.parent;
        u.keep = g.keep;
        u.add = g.add;
        u.copy_from = g.copy_from;
        u.copy_to = g.copy_to;
        u.copy_slots = g.copy_slots;
        DeviceScope scope(h->device);
        cuda_check(nut::pages_update(u, static_cast<cudaStream_t>(stream)), "pages update");
    });
}

nut_status nut_beam_create(int64_t sequences, int64_t beams, int64_t vocab, int64_t n_out, int device, nut_beam **out) {
    return guarded([&] {
        if (!out)
            refuse(NUT_INVALID_ARGUMENT, "beam", "null argument");
        *out = nullptr;
        if (sequences <= 0 || beams <= 0 || vocab <= 0 || n_out <= 0)
            refuse(NUT_INVALID_ARGUMENT, "beam", "invalid dimensions");
        if (n_out > NUT_BEAM_MAX_OUT)
            refuse(NUT_LENGTH_ERROR, "beam", "n_out exceeds NUT_BEAM_MAX_OUT");
        if (sequences > kMostRows || beams > 1024 || sequences * beams > kMostRows || vocab > (1 << 28))
            refuse(NUT_LENGTH_ERROR, "beam", "dimensions exceed device limits");
        /* a row's first tile may begin up to 7 elements before it.  Runs for some 16
         * warps on every SM: with fewer its memory waits, more warps list and reduce more, of which n_out
         * is the measure.  With 12, 14, 16, 18, 20, 24 and 28, us in a graph:
         *   64 rows of 128,000, fp32, of 16    25.7   26.4   26.4   26.4   28.1   28.2   32.8
         *   256 of 128,000, fp32, of 16        45.5   44.7   43.3   44.5   44.0   44.0   49.4
         *   256 of 128,000, fp32, of 64        98.9  110.8  106.2  118.5  117.5  128.3  145.8
         *   1,024 of 32,000, fp32, of 16       54.0   45.8   45.8   45.8   45.8   43.5   49.0
         *   256 of 32,000, bf16, of 16         24.1   23.3   23.3   23.3   22.3   22.3   23.3
         *   512 of 128,000, bf16, of 16        68.4   64.8   64.8   63.7   63.7   62.2   58.4
         * (up to 32 rows are a run a tile: no difference) */
        const int64_t tiles = (vocab + 7 + nut::kBeamTile - 1) / nut::kBeamTile, rows = sequences * beams;
        if (rows * tiles > INT_MAX / NUT_BEAM_MAX_OUT)
            refuse(NUT_LENGTH_ERROR, "beam", "dimensions exceed device limits");
        DeviceScope scope(device);
        int sms = 0;
        cuda_check(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device), "count SMs");
        const int64_t wanted = std::min(tiles, std::max<int64_t>(1, (16 * sms) / rows));
        const int64_t run_tiles = (tiles + wanted - 1) / wanted, runs = (tiles + run_tiles - 1) / run_tiles;
        auto h = std::make_unique<nut_beam>();
        h->device = device;
        nut::BeamSelect &b = h->b;
        b.sequences = int(sequences);
        b.beams = int(beams);
        b.vocab = int(vocab);
        b.n_out = int(n_out);
        b.runs = int(runs);
        b.run_tiles = int(run_tiles);
        Workspace &w = h->space;
        const size_t all = size_t(rows * runs);
        const size_t parts = w.part(all, sizeof(nut::BeamPart)), best = w.part(all * size_t(n_out), 8);
        w.make(device, 0);
        b.parts = reinterpret_cast<nut::BeamPart *>(w.block + parts);
        b.best = reinterpret_cast<unsigned long long *>(w.block + best);
        *out = h.release();
    });
}

nut_status nut_beam_destroy(nut_beam *h) {
    return guarded([&] {
        if (!h)
            return;
        DeviceScope scope(h->device);
        delete h;
    });
}

nut_status nut_beam_select(nut_beam *h, const nut_beam_select_args *args, void *stream) {
    return guarded([&] {
        if (!h || !args)
            refuse(NUT_INVALID_ARGUMENT, "beam", "null argument");
        const nut_beam_select_args &g = *args;
        nut::BeamSelect b = h->b;
        if (!g.logits || !g.scores || !g.out_scores || !g.out_rows || !g.out_tokens)
            refuse(NUT_INVALID_ARGUMENT, "beam", "null logits, scores or outputs");
        if (g.type != NUT_F32 && g.type != NUT_F16 && g.type != NUT_BF16)
            refuse(NUT_INVALID_ARGUMENT, "beam", "unknown type of logits");
        if (reinterpret_cast<uintptr_t>(g.logits) % (g.type == NUT_F32 ? 4 : 2) != 0)
            refuse(NUT_INVALID_ARGUMENT, "beam", "logits must be a multiple of their element");
        if (g.logits_stride != 0 && g.logits_stride < b.vocab)
            refuse(NUT_INVALID_ARGUMENT, "beam", "logits_stride is less than a row");
        if (g.sequences < 0)
            refuse(NUT_INVALID_ARGUMENT, "beam", "negative sequence count");
        if (g.sequences > b.sequences)
            refuse(NUT_LENGTH_ERROR, "beam", "more sequences than created for");
        if (g.eos < -1 || g.eos >= b.vocab)
            refuse(NUT_INVALID_ARGUMENT, "beam", "eos outside the vocabulary");
        if (g.finished && g.eos < 0)
            refuse(NUT_INVALID_ARGUMENT, "beam", "finished beams need eos");
        if (!aligned4({g.scores, g.out_scores, g.out_rows, g.out_tokens}))
            refuse(NUT_INVALID_ARGUMENT, "beam", "arrays must be multiples of their elements");
        if (g.sequences == 0)
            return;
        /* a request's outputs are written while others' beams are still read */
        if (b.n_out != b.beams && (g.out_scores == g.scores || (g.finished && g.out_finished == g.finished)))
            refuse(NUT_INVALID_ARGUMENT, "beam", "outputs in the inputs' place need n_out to be beams");
        b.logits = g.logits;
        b.stride = g.logits_stride ? g.logits_stride : b.vocab;
        b.scores = g.scores;
        b.finished = g.finished;
        b.out_scores = g.out_scores;
        b.out_rows = g.out_rows;
        b.out_tokens = g.out_tokens;
        b.out_finished = g.out_finished;
        b.sequences = int(g.sequences);
        b.eos = g.eos;
        b.type = g.type;
        DeviceScope scope(h->device);
        cuda_check(nut::beam_select(b, static_cast<cudaStream_t>(stream)), "beam select");
    });
}

} // extern "C"
