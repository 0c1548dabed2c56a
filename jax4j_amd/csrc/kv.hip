// The 8-bit key/value cache, host side: which sequence holds which pages, the checks of every call, and what is launched
// (layout and kernels: kv.h). Engine-local; the reference has no attention.
//
// Pages, lengths and reference counts live here, so a call that cannot be served (no page left, a table full, a mask that
// would look at freed tokens) is refused before anything is enqueued or changed. The device has the tables and the current
// step (which sequences, their lengths and rows), which a kernel with the changes in its arguments keeps up, in stream order.
// A page is taken lowest first. A call takes the host memory that it needs before it changes anything, so that one that finds
// none leaves the cache as it was; a cache whose change the device did not get (a launch failed) is refused from then on.
#include <limits.h>
#include <math.h>

#include <algorithm>
#include <exception>
#include <memory>
#include <vector>

#include "engine.h"
#include "kept_memory.h"
#include "kv.h"

namespace j4q {
namespace {

// Rows of partial results that a cache has room for: (D + 2) floats each.
constexpr int64_t kPartRows = 65536;
// Query rows (tokens x group) of a sequence and kv head up to which the kernel for few rows runs, which reads the cache once for
// 8 rows, and that for some rows (32; heads up to 128, whose rows fit the registers). 8 kv heads of 128, fp32, the one and the
// other: 16 rows of 500 tokens 9.8 and 12.1 us, of 8000 in 64 sequences 234 and 198; 20 rows 9.9 and 12.7, 313 and 200. Up to 16 the
// short ones decide, and that a bf16 result comes of fp32 weights. Some rows and many: 32 rows of 8000 tokens in 64 sequences 203
// us and 372, into bf16 186 and 220; of 500 in one 13.6 and 12.5, 12.5 and 11.5.
constexpr int kFewRows = 16, kSomeRows = 32;

struct Seq {
    int64_t len = 0;
    std::vector<int32_t> pages;  // -1: evicted
    // pages of no token outside [gone0, gone1) have been evicted
    int64_t gone0 = 0, gone1 = 0;
};

struct Kv {
    j4q_kv_config c{};
    uint32_t gen = 0;
    bool live = false;
    int64_t page_bytes = 0, layer_bytes = 0;
    int block_shift = 0;
    uint8_t *pool = nullptr;
    int32_t *words = nullptr;  // tables, then the step: seq, len, row0, block0
    float *part = nullptr;
    uint64_t bytes = 0;
    std::vector<Seq> seqs;
    std::vector<int32_t> refs;
    std::vector<uint64_t> free_bits;
    int64_t free_pages = 0, hint = 0;  // no free page below 64 hint
    // the current step
    std::vector<int32_t> step_seq, step_tokens;
    int32_t step_rows = 0, step_blocks = 0, step_most_blocks = 0;
    bool step_checked = false;
    // calls on one stream after another
    hipEvent_t done = nullptr;
    hipStream_t last = nullptr;
    bool used = false;
    bool lost = false;  // the device's words are not what is here

    int32_t at_seq() const { return c.sequences * c.sequence_pages; }
    int32_t at_len() const { return at_seq() + c.sequences; }
    int32_t at_row0() const { return at_len() + c.sequences; }
    int32_t at_block0() const { return at_row0() + c.sequences + 1; }
    int64_t word_count() const { return (int64_t)c.sequences * (c.sequence_pages + 4) + 2; }

    int32_t take() {
        while (!free_bits[(size_t)hint]) hint++;
        uint64_t &w = free_bits[(size_t)hint];
        const int b = __builtin_ctzll(w);
        w &= w - 1;
        free_pages--;
        const int32_t p = (int32_t)(64 * hint + b);
        refs[(size_t)p] = 1;
        return p;
    }
    void drop(int32_t p) {
        if (p < 0 || --refs[(size_t)p] > 0) return;
        free_bits[(size_t)(p / 64)] |= 1ull << (p % 64);
        free_pages++;
        hint = std::min<int64_t>(hint, p / 64);
    }
    KvLayer layer(int32_t l) const {
        KvLayer k;
        k.base = pool + l * layer_bytes;
        k.page_bytes = page_bytes;
        k.scales = (int32_t)(c.kv_heads * (c.page_tokens / kKvBlock)) * 2 * kKvBlock * c.head_dim;
        k.kv_heads = c.kv_heads;
        k.dim = c.head_dim;
        k.block_shift = block_shift;
        return k;
    }
    KvStep step() const {
        KvStep s;
        s.table = words;
        s.seq = words + at_seq();
        s.len = words + at_len();
        s.row0 = words + at_row0();
        s.block0 = words + at_block0();
        s.sequence_pages = c.sequence_pages;
        s.n = (int32_t)step_seq.size();
        s.rows = step_rows;
        return s;
    }
};

std::vector<std::unique_ptr<Kv>> g_kvs;

Kv *lookup(j4q_kv h) {
    const uint64_t lo = h & 0xffffffffu;
    if (lo == 0 || lo > g_kvs.size()) return nullptr;
    Kv *k = g_kvs[lo - 1].get();
    return k->live && k->gen == (uint32_t)(h >> 32) ? k : nullptr;
}

int get(j4q_kv h, const char *op, Kv **out, bool lost_too = false) {
    *out = lookup(h);
    if (!*out) return report_error(J4Q_EHANDLE, "%s: unknown or destroyed cache 0x%llx", op, (unsigned long long)h);
    if ((*out)->lost && !lost_too) return report_error(J4Q_EHIP, "%s: an earlier call on this cache failed on the device", op);
    return J4Q_OK;
}

// What an entry point answers where host memory ran out in it.
int no_memory(const char *op) { return report_error(J4Q_ENOMEM, "%s failed: out of host memory", op); }

bool aligned(const void *p, uintptr_t a) { return ((uintptr_t)p & (a - 1)) == 0; }

// One call's launches on its stream, behind the cache's last call. That one's last launch has completed k.done, but on the engine
// stream, which outlives the cache: there calls follow one another, and the event is recorded only when a call leaves it (a launch
// with an event takes the host 1 to 2 us more). Every other handle may have named another stream before (that of another
// thread, one destroyed since), so an equal one saves the wait only where nothing is left to wait for (0.3 us of the host's
// time a call to ask and to wait). Under capture the caller orders the graph's launches.
struct Call {
    Kv &k;
    hipStream_t s;
    bool captured, behind = true;
    hipError_t e;

    Call(Kv &kv, void *stream) : k(kv), s(stream ? (hipStream_t)stream : abi::stream()) {
        hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
        e = hipStreamIsCapturing(s, &st);
        captured = st != hipStreamCaptureStatusNone;
    }
    bool from_engine() const { return k.used && k.last == abi::stream() && s != k.last; }
    // Before anything changes: whether the call can go out on its stream. capture: why a captured graph cannot hold it, or nullptr.
    int check(const char *op, const char *capture) const {
        if (e != hipSuccess) {  // neither kind of call: the one would wait for nothing, the other be a graph's
            (void)hipGetLastError();
            return report_hip(op, e);
        }
        if (captured) return capture ? report_error(J4Q_EINVAL, "%s: %s", op, capture) : J4Q_OK;
        if (from_engine() && capturing(abi::stream()))  // an event recorded there now would draw this call into the graph
            return report_error(J4Q_EINVAL, "%s: another stream cannot wait for the cache's last call while the engine stream, where that is, is captured", op);
        return J4Q_OK;
    }
    // Before the first launch.
    void order() {
        if (captured || !k.used) return;
        if (from_engine()) e = hipEventRecord(k.done, k.last);
        else if (s == k.last && (s == abi::stream() || completed(k.done))) return;
        if (e == hipSuccess) e = hipStreamWaitEvent(s, k.done, 0);
        behind = e == hipSuccess;
    }
    bool recorded() const { return !captured && s != abi::stream(); }
    hipEvent_t event(bool last) const { return last && recorded() ? k.done : nullptr; }
    int end_change(const char *op) {
        k.lost |= e != hipSuccess;
        return end(op);
    }
    int end(const char *op) {
        if (!behind) {  // nothing went out, and the call before is still what the next one waits for
            (void)hipGetLastError();  // a launch checks for errors by the last one
            return report_hip(op, e);
        }
        if (e != hipSuccess && recorded()) (void)hipEventRecord(k.done, s);
        if (!captured) {
            k.last = s;
            k.used = true;
        }
        return e == hipSuccess ? J4Q_OK : report_hip(op, e);
    }
};

// Changes of the device's words, merged where they go on by equal steps.
struct Changes {
    std::vector<KvRun> runs;
    void add(int64_t at, int32_t value) {
        if (!runs.empty()) {
            KvRun &r = runs.back();
            if (r.at + r.count == at && (r.count == 1 || r.value + (int64_t)r.step * r.count == value)) {
                const int64_t step = (int64_t)value - r.value;
                if (r.count > 1 || (step >= INT_MIN && step <= INT_MAX)) {
                    if (r.count == 1) r.step = (int32_t)step;
                    r.count++;
                    return;
                }
            }
        }
        runs.push_back(KvRun{(int32_t)at, value, 0, 1});
    }
    // last: nothing follows in the call.
    void launch(Call &c, bool last) const {
        for (size_t at = 0; at < runs.size() && c.e == hipSuccess; at += kKvRuns) {
            KvRuns r;
            r.words = c.k.words;
            r.n = (int32_t)std::min<size_t>(kKvRuns, runs.size() - at);
            std::copy_n(runs.begin() + (long)at, r.n, r.run);
            c.e = launch_kv_runs(r, c.s, c.event(last && at + kKvRuns >= runs.size()));
        }
    }
};

using Pairs = std::vector<std::pair<int32_t, int32_t>>;  // page, its copy

void copy_pages(Call &c, const Pairs &pairs, bool last) {
    for (size_t at = 0; at < pairs.size() && c.e == hipSuccess; at += kKvPairs) {
        KvPairs p;
        p.pool = c.k.pool;
        p.page_bytes = c.k.page_bytes;
        p.layer_bytes = c.k.layer_bytes;
        p.layers = c.k.c.layers;
        p.n = (int32_t)std::min<size_t>(kKvPairs, pairs.size() - at);
        for (int i = 0; i < p.n; i++) p.src[i] = pairs[at + (size_t)i].first, p.dst[i] = pairs[at + (size_t)i].second;
        c.e = launch_kv_copy(p, c.s, c.event(last && at + kKvPairs >= pairs.size()));
    }
}

int check_seqs(const Kv &k, const char *op, const int32_t *seqs, int32_t n, bool unique) {
    if (n < 1 || n > k.c.sequences || !seqs) return report_error(J4Q_EINVAL, "%s: %d sequences, of a cache of %d", op, n, k.c.sequences);
    std::vector<bool> seen((size_t)k.c.sequences);
    for (int32_t i = 0; i < n; i++) {
        if (seqs[i] < 0 || seqs[i] >= k.c.sequences)
            return report_error(J4Q_EINVAL, "%s: sequence %d out of range [0, %d)", op, seqs[i], k.c.sequences);
        if (unique && seen[(size_t)seqs[i]]) return report_error(J4Q_EINVAL, "%s: sequence %d twice", op, seqs[i]);
        seen[(size_t)seqs[i]] = true;
    }
    return J4Q_OK;
}

// What a replayed graph cannot do: it would repeat changes that the host has made once.
constexpr char kChanges[] = "changes the cache's pages, which a captured graph cannot repeat";

void end_step(Kv &k) {
    k.step_seq.clear();
    k.step_tokens.clear();
    k.step_rows = 0;
}
bool in_step(const Kv &k, int32_t seq) { return std::find(k.step_seq.begin(), k.step_seq.end(), seq) != k.step_seq.end(); }

// The last tokens[i] tokens of seqs[i] as the current step (lengths as they are now): at most step_changes(n) runs.
size_t step_changes(int32_t n) { return 4 * (size_t)n + 2; }
void set_step(Kv &k, const int32_t *seqs, const int32_t *tokens, int32_t n, Changes *ch) {
    k.step_seq.assign(seqs, seqs + n);
    k.step_tokens.assign(tokens, tokens + n);
    k.step_checked = false;
    k.step_most_blocks = 0;
    for (int32_t i = 0; i < n; i++) ch->add(k.at_seq() + i, seqs[i]);
    for (int32_t i = 0; i < n; i++) ch->add(k.at_len() + i, (int32_t)k.seqs[(size_t)seqs[i]].len);
    int32_t rows = 0;
    ch->add(k.at_row0(), 0);
    for (int32_t i = 0; i < n; i++) ch->add(k.at_row0() + i + 1, rows += tokens[i]);
    int32_t blocks = 0;
    ch->add(k.at_block0(), 0);
    for (int32_t i = 0; i < n; i++) {
        const int64_t len = k.seqs[(size_t)seqs[i]].len;
        const int32_t b = (int32_t)((len - 1) / kKvBlock - (len - tokens[i]) / kKvBlock + 1);
        k.step_most_blocks = std::max(k.step_most_blocks, b);
        ch->add(k.at_block0() + i + 1, blocks += b);
    }
    k.step_rows = rows;
    k.step_blocks = blocks;
}

int check_rows(const char *op, const int32_t *tokens, int32_t n) {
    int64_t rows = 0;
    for (int32_t i = 0; i < n; i++) {
        if (tokens[i] < 1) return report_error(J4Q_EINVAL, "%s: %d tokens of sequence %d of the step (at least one)", op, tokens[i], i);
        rows += tokens[i];
    }
    if (rows > 1 << 24) return report_error(J4Q_EUNSUPPORTED, "%s: %lld tokens in a step (at most %d)", op, (long long)rows, 1 << 24);
    return J4Q_OK;
}

int fill_rope(const char *op, const j4q_rope *r, int32_t head_dim, int64_t rows, bool positions, KvRope *out) {
    *out = KvRope{};
    if (!r) return J4Q_OK;
    if (!r->cos_table || !r->sin_table || r->table_rows < 1 || r->table_rows > INT_MAX)
        return report_error(J4Q_EINVAL, "%s: rotary positions need tables of 1 to 2^31 - 1 rows", op);
    if (r->dims < 2 || r->dims % 2 || r->dims > head_dim || r->dims > kKvMaxDim)
        return report_error(J4Q_EINVAL, "%s: %d rotary channels of a head of %d (an even number, at most %d)", op, r->dims, head_dim, std::min(head_dim, kKvMaxDim));
    if (!aligned(r->cos_table, 4) || !aligned(r->sin_table, 4) || !aligned(r->positions, 4))
        return report_error(J4Q_EINVAL, "%s: rotary tables and positions must be 4-byte aligned", op);
    if (!r->positions && positions) return report_error(J4Q_EINVAL, "%s: positions is NULL", op);
    int axes = 1;
    if (r->pair_axis)
        for (int i = 0; i < r->dims / 2; i++) {
            out->axis[i] = r->pair_axis[i];
            axes = std::max(axes, r->pair_axis[i] + 1);
        }
    if (axes > 1 && !r->positions) return report_error(J4Q_EINVAL, "%s: pairs of %d axes need positions", op, axes);
    out->cos = r->cos_table;
    out->sin = r->sin_table;
    out->positions = r->positions;
    out->table_rows = (int32_t)r->table_rows;
    out->pairs = r->dims / 2;
    out->axes = axes;
    out->interleaved = r->interleaved != 0;
    out->rows = (int32_t)rows;
    return J4Q_OK;
}

bool dense_type(int t) { return t == J4Q_KIND_F32 || t == J4Q_KIND_BF16; }

// Row strides in elements (0: rows lie one behind the other), rows of 16-byte pieces.
int check_stride(const char *op, const char *what, const void *p, int type, int64_t width, int64_t *stride) {
    const int64_t e = type == J4Q_KIND_BF16 ? 2 : 4;
    if (!*stride) *stride = width;
    if (!aligned(p, 16) || *stride < width || *stride * e % 16 != 0 || *stride > (1ll << 40))
        return report_error(J4Q_EINVAL, "%s: %s must be 16-byte aligned, its rows %lld values or more apart, a multiple of 16 bytes", op, what, (long long)width);
    return J4Q_OK;
}

// Whether two tensors of rows `width` bytes wide share a byte.
bool overlap(const void *a, int64_t a_stride, int64_t a_width, const void *b, int64_t b_stride, int64_t b_width, int64_t rows) {
    const uintptr_t a0 = (uintptr_t)a, b0 = (uintptr_t)b;
    if (a0 >= b0 + (rows - 1) * b_stride + b_width || b0 >= a0 + (rows - 1) * a_stride + a_width) return false;
    if (a_stride != b_stride) return true;
    const int64_t between = (int64_t)(b0 - a0) % a_stride, at = between < 0 ? between + a_stride : between;  // windows of the same rows
    return at < a_width || at + b_width > a_stride;
}

// Tiles of 64 tokens that the workgroups of a call's sequences walk for one kv head: all of them, the longest walk's, and how many
// workgroups and rows there are.
struct Walks {
    int64_t tiles = 0, most = 0, groups = 0, rows = 0;
};
Walks walks_of(const Kv &k, const KvAttend &a) {
    Walks w;
    for (size_t i = 0; i < k.step_seq.size(); i++) {
        const int64_t before = k.seqs[(size_t)k.step_seq[i]].len - k.step_tokens[i], rows = (int64_t)k.step_tokens[i] * a.group;
        if (rows < a.rows_from || rows > a.rows_to) continue;
        w.rows += rows;
        w.groups += (rows + a.row_tile - 1) / a.row_tile;
        for (int64_t r = 0; r < rows; r += a.row_tile) {
            const int64_t last = std::min(rows, r + a.row_tile) - 1;
            const int64_t count = kv_tiles((int)(before + r / a.group), (int)(before + last / a.group), a.window, a.sinks).count();
            w.tiles += count;
            w.most = std::max(w.most, count);
        }
    }
    return w;
}
// Cuts walks of up to `most` tiles into ranges of split_tiles, as far as there is room for their parts. A graph's later runs may
// have longer ones.
void set_splits(const Kv &k, bool captured, int64_t most, int64_t split_tiles, KvAttend *a) {
    const int64_t room = kPartRows / ((int64_t)k.step_seq.size() * k.c.kv_heads * a->max_rows);
    const int64_t longest = captured && most > 0 ? std::max(most, ((int64_t)k.c.sequence_pages * k.c.page_tokens + kKvTile - 1) / kKvTile) : most;
    a->splits = (int32_t)std::max<int64_t>(1, std::min<int64_t>({(longest + split_tiles - 1) / split_tiles, room, kKvSplits}));
    a->split_tiles = (int32_t)std::max(split_tiles, (most + a->splits - 1) / a->splits);
}

// One range up to `alone` tiles, or up to `half` where half of the CUs have a workgroup; else ranges of four or more that fill the CUs
// once.
void split_filled(const Kv &k, bool captured, int64_t alone, int64_t half, KvAttend *a) {
    constexpr int64_t kFilled = 256, kLeast = 4;
    const Walks w = walks_of(k, *a);
    if (w.groups * k.c.kv_heads >= kFilled / 2) alone = half;
    set_splits(k, captured, w.most, std::max(w.most <= alone ? alone : kLeast, (w.tiles * k.c.kv_heads + kFilled - 1) / kFilled), a);
}

// Few rows: one workgroup of a CU's registers each, so ranges where the rows alone leave CUs idle. Joining them costs 4 to 5 us, a
// round of the 8 waves over a tile each 2.4, and less where only four of them have one, alone on their SIMDs (one request, 8 kv
// heads of 128: 11 tiles 10.0 us in one range, 10.7 in three; 16 tiles 11.3, and 13.2 in two; heads of 64 7.7, 9.2 in four; 32
// tiles 16.2, 12.7 in four, 11.2 in eight; 128 tiles 46, 14.0 in sixteen, 12.9 in thirty-two). Half of the CUs are better left idle
// for up to 32 tiles (16 requests, 32 tiles in one range and in two: heads of 64 11.8 us and 13.6, of 96 13.9 and 15.6, of 128 19.1
// and 21.9, of 192 22.4 and 26.1; heads of 128, 64 tiles 35.3 and 34.7). Heads of 256, whose four waves have twice the bytes a
// tile, are cut sooner (one request, in one range and in ranges of four: 8 tiles 13.5 and 14.5, 12 tiles 16.0 and 14.7, 16 tiles
// 18.4 and 14.8; 16 requests, in one and in two: 24 tiles 27.3 and 28.4, 32 tiles 33.8 to 35.0 and 33.6 to 33.8).
void split_few(const Kv &k, bool captured, KvAttend *a) {
    a->row_tile = a->max_rows <= 4 ? 4 : 8;
    if (k.c.head_dim > 192) split_filled(k, captured, 8, 24, a);
    else split_filled(k, captured, 16, 32, a);
}

// Some rows: a workgroup is a CU's as well, whose 8 waves take a tile each in a round; ranges of 4 tiles beside each other where
// there are workgroups to spare (one request, 24 rows of 8 kv heads of 128: 16 tiles 13.5 us in four ranges, 14.1 in one; 63
// tiles 14.8 in ranges of 4, 15.6 of 8 and 17.7 of 16; 16 requests, 32 tiles in one range and in two: heads of 64 14.2 and 15.7, of
// 96 16.4 and 18.5, of 128 20.7 and 23.2).
void split_some(const Kv &k, bool captured, KvAttend *a) {
    a->row_tile = 32;
    split_filled(k, captured, 8, 32, a);
}

// Many rows: workgroups of 256, whose conversion of a tile serves the most rows, or of 128, two to a CU, which fill the chip sooner:
// 8 kv heads of 128 with 4 query heads each, into bf16, a chunk of 512 tokens behind 3584 (64 workgroups of 256) 55 us and with 128
// 67, the last 64 tokens of 4096 (8) 30 and 26; a prompt of 2048, whose workgroups walk 1 to 32 tiles (256) 70 and 65, one of
// 8192 (1024) 561 and 602.
// Ranges by what they are estimated to cost: a tile takes a workgroup 1.3 us (of 128 rows), the chip's throughput has a floor,
// and parts are written and read back, behind a launch. (The last 64 tokens of 4096, one kv head: 33.4 us in 4 ranges, 17.8 in 16.)
void split_many(const Kv &k, bool captured, KvAttend *a) {
    const double heads = k.c.kv_heads, width = k.c.head_dim / 128.0;
    a->row_tile = 256;
    int64_t groups = 0;
    for (size_t i = 0; i < k.step_seq.size(); i++) {
        const int64_t rows = (int64_t)k.step_tokens[i] * a->group;
        if (rows >= a->rows_from && rows <= a->rows_to) groups += (rows + 255) / 256;
    }
    a->splits = 1;
    a->split_tiles = INT_MAX / 2;
    // rows that one workgroup of 128 holds (64 rows of 8000 tokens in 64 sequences: 277 us, of 256 with empty waves 519)
    const bool wide = k.c.head_dim <= 128 && a->max_rows > 128;
    if (wide && groups * k.c.kv_heads >= 448) return;
    Walks w = walks_of(k, *a);
    if (!wide || groups * k.c.kv_heads < 64 || 4 * w.tiles < 3 * w.most * w.groups) {
        a->row_tile = 128;
        if (groups * k.c.kv_heads >= 448) return;
        w = walks_of(k, *a);
    }
    const double tile_us = (a->row_tile == 256 ? 1.55 : 1.3) * width, all_us = (a->row_tile == 256 ? 1.9 : 0.9) * width * (double)w.tiles * heads / 256;
    double best = 0;
    int64_t ranges = 1;
    for (int64_t s = 1; s <= 64 && s <= w.most; s++) {
        const double walk = tile_us * (double)((w.most + s - 1) / s);
        const double join = s == 1 ? 0 : (s > 16 ? 8 : 4) + (double)w.rows * heads * (double)s * 4 * k.c.head_dim / 4.5e6;
        const double us = std::max(walk, all_us) + join;
        if (s == 1 || us < best) best = us, ranges = s;
    }
    set_splits(k, captured, w.most, (w.most + ranges - 1) / ranges, a);
    if (ranges == 1 && !captured) a->splits = 1;
}

}  // namespace
}  // namespace j4q

using namespace j4q;

extern "C" {

int j4q_kv_create(const j4q_kv_config *config, j4q_kv *out) try {
    if (!config || !out) return report_error(J4Q_EINVAL, "kv cache: NULL argument");
    const j4q_kv_config c = *config;
    if (c.layers < 1 || c.layers > 65535 || c.kv_heads < 1 || c.kv_heads > 1024)
        return report_error(J4Q_EINVAL, "kv cache: %d layers, %d kv heads out of range [1, 65535], [1, 1024]", c.layers, c.kv_heads);
    if (c.head_dim != 64 && c.head_dim != 96 && c.head_dim != 128 && c.head_dim != 192 && c.head_dim != 256)
        return report_error(J4Q_EUNSUPPORTED, "kv cache: head_dim %d (64, 96, 128, 192 or 256)", c.head_dim);
    if (c.page_tokens != 16 && c.page_tokens != 32 && c.page_tokens != 64)
        return report_error(J4Q_EUNSUPPORTED, "kv cache: pages of %d tokens (16, 32 or 64)", c.page_tokens);
    if (c.pages < 1 || c.pages > INT_MAX || c.sequences < 1 || c.sequence_pages < 1 ||
        (int64_t)c.sequence_pages * c.page_tokens > 1 << 30 || (int64_t)c.sequences * (c.sequence_pages + 4ll) + 2 > INT_MAX)
        return report_error(J4Q_EINVAL, "kv cache: %lld pages, %d sequences of %d pages out of range", (long long)c.pages, c.sequences, c.sequence_pages);
    const int64_t page = kv_page_bytes(c.kv_heads, c.head_dim, c.page_tokens);
    if (c.pages > INT64_MAX / page / c.layers)
        return report_error(J4Q_EINVAL, "kv cache: %lld pages of %lld bytes in %d layers", (long long)c.pages, (long long)page, c.layers);
    std::lock_guard<std::mutex> lk(abi::lock());
    int rc = abi::ready_locked();
    if (rc) return rc;
    if (capturing(abi::stream())) return report_error(J4Q_EINVAL, "kv cache: %s", kChanges);
    std::unique_ptr<Kv> k(new Kv);
    g_kvs.reserve(g_kvs.size() + 1);
    k->seqs.resize((size_t)c.sequences);
    k->refs.assign((size_t)c.pages, 0);
    k->free_bits.assign((size_t)((c.pages + 63) / 64), ~0ull);
    k->step_seq.reserve((size_t)c.sequences);
    k->step_tokens.reserve((size_t)c.sequences);
    k->c = c;
    k->page_bytes = page;
    k->layer_bytes = page * c.pages;
    k->block_shift = c.page_tokens == 64 ? 2 : c.page_tokens == 32 ? 1 : 0;
    const uint64_t pool = (uint64_t)(k->layer_bytes * c.layers), words = align256((uint64_t)k->word_count() * 4),
                   part = (uint64_t)(kPartRows * (c.head_dim + 2)) * 4;
    hipError_t e = abi::malloc_locked((void **)&k->pool, pool);
    if (e == hipSuccess) e = abi::malloc_locked((void **)&k->words, words);
    if (e == hipSuccess) e = abi::malloc_locked((void **)&k->part, part);
    if (e == hipSuccess) e = hipEventCreateWithFlags(&k->done, hipEventDisableTiming | hipEventDisableSystemFence);
    if (e == hipSuccess) {
        KvRuns r;
        r.words = k->words;
        r.n = 1;
        r.run[0] = KvRun{0, -1, 0, (int32_t)k->word_count()};
        e = launch_kv_runs(r, abi::stream(), nullptr);
    }
    if (e != hipSuccess) {
        (void)hipGetLastError();
        if (k->done) (void)hipEventDestroy(k->done);
        for (void *p : {(void *)k->pool, (void *)k->words, (void *)k->part})
            if (p) (void)hipFree(p);
        return report_hip("kv cache", e);
    }
    k->last = abi::stream();
    k->used = true;
    k->bytes = pool + words + part;
    if (c.pages % 64) k->free_bits.back() = (1ull << (c.pages % 64)) - 1;
    k->free_pages = c.pages;
    k->live = true;
    size_t slot = 0;
    while (slot < g_kvs.size() && g_kvs[slot]->live) slot++;
    k->gen = slot < g_kvs.size() ? g_kvs[slot]->gen + 1 : 1;
    const j4q_kv handle = ((uint64_t)k->gen << 32) | (uint64_t)(slot + 1);
    if (slot == g_kvs.size()) g_kvs.push_back(std::move(k));
    else g_kvs[slot] = std::move(k);
    *out = handle;
    return J4Q_OK;
} catch (const std::exception &) {
    return no_memory("kv cache");
}

int j4q_kv_destroy(j4q_kv kv) {
    if (kv == 0) return J4Q_OK;
    std::lock_guard<std::mutex> lk(abi::lock());
    Kv *k;
    int rc = get(kv, "kv destroy", &k, true);
    if (rc) return rc;
    if ((rc = abi::ready_locked())) return rc;
    const hipError_t e = hipDeviceSynchronize();  // calls may still run on any stream
    if (e != hipSuccess) return report_hip("kv destroy", e);
    (void)hipEventDestroy(k->done);
    (void)hipFree(k->pool);
    (void)hipFree(k->words);
    (void)hipFree(k->part);
    const uint32_t gen = k->gen;
    *k = Kv();
    k->gen = gen;
    return J4Q_OK;
}

int j4q_kv_info(j4q_kv kv, j4q_kv_desc *out) {
    if (!out) return report_error(J4Q_EINVAL, "kv info: out is NULL");
    std::lock_guard<std::mutex> lk(abi::lock());
    Kv *k;
    const int rc = get(kv, "kv info", &k, true);
    if (rc) return rc;
    *out = j4q_kv_desc{};
    out->config = k->c;
    out->pages_free = k->free_pages;
    out->bytes = k->bytes;
    out->page_bytes = (uint64_t)k->page_bytes;
    out->step_sequences = (int32_t)k->step_seq.size();
    out->step_rows = k->step_rows;
    return J4Q_OK;
}

int j4q_kv_tables(j4q_kv kv, const int32_t *seqs, int32_t n, int64_t *lengths, int32_t *pages, int32_t capacity) try {
    std::lock_guard<std::mutex> lk(abi::lock());
    Kv *k;
    int rc = get(kv, "kv tables", &k);
    if (rc) return rc;
    if ((rc = check_seqs(*k, "kv tables", seqs, n, false))) return rc;
    if (capacity < 0 || (capacity > 0 && !pages)) return report_error(J4Q_EINVAL, "kv tables: room for %d pages", capacity);
    for (int32_t i = 0; i < n; i++) {
        const Seq &q = k->seqs[(size_t)seqs[i]];
        if (lengths) lengths[i] = q.len;
        const size_t have = std::min(q.pages.size(), (size_t)capacity);
        int32_t *to = pages + (int64_t)i * capacity;
        std::copy_n(q.pages.begin(), have, to);
        std::fill(to + have, to + capacity, -1);
    }
    return J4Q_OK;
} catch (const std::exception &) {
    return no_memory("kv tables");
}

int j4q_kv_extend(j4q_kv kv, const int32_t *seqs, const int32_t *tokens, int32_t n, void *stream) try {
    std::lock_guard<std::mutex> lk(abi::lock());
    Kv *k;
    int rc = get(kv, "kv extend", &k);
    if (rc) return rc;
    if (!tokens) return report_error(J4Q_EINVAL, "kv extend: tokens is NULL");
    if ((rc = check_seqs(*k, "kv extend", seqs, n, true)) || (rc = check_rows("kv extend", tokens, n))) return rc;
    const int64_t per = k->c.page_tokens;
    int64_t need = 0;
    std::vector<int32_t> left;  // references to a shared, partly filled page, once the sequences before have their own
    std::vector<int32_t> shared;
    for (int32_t i = 0; i < n; i++) {
        const Seq &q = k->seqs[(size_t)seqs[i]];
        const int64_t pages = (q.len + tokens[i] + per - 1) / per;
        if (pages > k->c.sequence_pages)
            return report_error(J4Q_EINVAL, "kv extend: sequence %d would hold %lld tokens, its table %lld", seqs[i], (long long)(q.len + tokens[i]),
                                (long long)(k->c.sequence_pages * per));
        need += pages - (int64_t)q.pages.size();
        if (q.len % per) {
            const int32_t p = q.pages.back();
            size_t j = 0;
            while (j < shared.size() && shared[j] != p) j++;
            if (k->refs[(size_t)p] > 1) {
                if (j == shared.size()) {
                    shared.push_back(p);
                    left.push_back(k->refs[(size_t)p]);
                }
                if (left[j] > 1) {
                    left[j]--;
                    need++;
                }
            }
        }
    }
    if (need > k->free_pages)
        return report_error(J4Q_ENOMEM, "kv extend failed: %lld pages needed, %lld free", (long long)need, (long long)k->free_pages);
    if ((rc = abi::ready_locked())) return rc;
    Call c(*k, stream);
    if ((rc = c.check("kv extend", kChanges))) return rc;
    Changes ch;
    Pairs pairs;
    ch.runs.reserve((size_t)need + step_changes(n));
    pairs.reserve(shared.empty() ? 0 : (size_t)n);
    for (int32_t i = 0; i < n; i++) {
        std::vector<int32_t> &pages = k->seqs[(size_t)seqs[i]].pages;
        const size_t count = (size_t)((k->seqs[(size_t)seqs[i]].len + tokens[i] + per - 1) / per);
        if (count > pages.capacity()) pages.reserve(std::max(count, std::min(2 * pages.capacity(), (size_t)k->c.sequence_pages)));
    }
    for (int32_t i = 0; i < n; i++) {
        Seq &q = k->seqs[(size_t)seqs[i]];
        const int64_t table = (int64_t)seqs[i] * k->c.sequence_pages;
        if (q.len % per && k->refs[(size_t)q.pages.back()] > 1) {  // others hold the page that the new tokens go to
            const int32_t was = q.pages.back();
            q.pages.back() = k->take();
            k->drop(was);
            pairs.emplace_back(was, q.pages.back());
            ch.add(table + (int64_t)q.pages.size() - 1, q.pages.back());
        }
        q.len += tokens[i];
        while ((int64_t)q.pages.size() * per < q.len) {
            q.pages.push_back(k->take());
            ch.add(table + (int64_t)q.pages.size() - 1, q.pages.back());
        }
    }
    set_step(*k, seqs, tokens, n, &ch);
    c.order();
    copy_pages(c, pairs, false);
    ch.launch(c, true);
    return c.end_change("kv extend");
} catch (const std::exception &) {
    return no_memory("kv extend");
}

int j4q_kv_begin(j4q_kv kv, const int32_t *seqs, const int32_t *tokens, int32_t n, void *stream) try {
    std::lock_guard<std::mutex> lk(abi::lock());
    Kv *k;
    int rc = get(kv, "kv begin", &k);
    if (rc) return rc;
    if (!tokens) return report_error(J4Q_EINVAL, "kv begin: tokens is NULL");
    if ((rc = check_seqs(*k, "kv begin", seqs, n, true)) || (rc = check_rows("kv begin", tokens, n))) return rc;
    for (int32_t i = 0; i < n; i++)
        if (tokens[i] > k->seqs[(size_t)seqs[i]].len)
            return report_error(J4Q_EINVAL, "kv begin: sequence %d has %lld tokens, not %d", seqs[i], (long long)k->seqs[(size_t)seqs[i]].len, tokens[i]);
    if ((rc = abi::ready_locked())) return rc;
    Call c(*k, stream);
    if ((rc = c.check("kv begin", kChanges))) return rc;
    Changes ch;
    ch.runs.reserve(step_changes(n));
    set_step(*k, seqs, tokens, n, &ch);
    c.order();
    ch.launch(c, true);
    return c.end_change("kv begin");
} catch (const std::exception &) {
    return no_memory("kv begin");
}

int j4q_kv_fork(j4q_kv kv, const int32_t *src, const int32_t *dst, int32_t n, int share, void *stream) try {
    std::lock_guard<std::mutex> lk(abi::lock());
    Kv *k;
    int rc = get(kv, "kv fork", &k);
    if (rc) return rc;
    if ((rc = check_seqs(*k, "kv fork", dst, n, true)) || (rc = check_seqs(*k, "kv fork", src, n, false))) return rc;
    int64_t need = 0;
    size_t entries = 0;
    std::vector<bool> made((size_t)k->c.sequences);
    for (int32_t i = 0; i < n; i++) {
        if (k->seqs[(size_t)dst[i]].len)
            return report_error(J4Q_EINVAL, "kv fork: sequence %d holds %lld tokens", dst[i], (long long)k->seqs[(size_t)dst[i]].len);
        made[(size_t)dst[i]] = true;
        entries += k->seqs[(size_t)src[i]].pages.size();
        if (!share)
            for (int32_t p : k->seqs[(size_t)src[i]].pages) need += p >= 0;
    }
    for (int32_t i = 0; i < n; i++)
        if (made[(size_t)src[i]]) return report_error(J4Q_EINVAL, "kv fork: sequence %d is made by this call and copied by it", src[i]);
    if (need > k->free_pages)
        return report_error(J4Q_ENOMEM, "kv fork failed: %lld pages needed, %lld free", (long long)need, (long long)k->free_pages);
    if ((rc = abi::ready_locked())) return rc;
    Call c(*k, stream);
    if ((rc = c.check("kv fork", kChanges))) return rc;
    Changes ch;
    Pairs pairs;
    ch.runs.reserve(entries);
    pairs.reserve((size_t)need);
    for (int32_t i = 0; i < n; i++) k->seqs[(size_t)dst[i]].pages.reserve(k->seqs[(size_t)src[i]].pages.size());
    for (int32_t i = 0; i < n; i++) {
        Seq &d = k->seqs[(size_t)dst[i]];
        d = k->seqs[(size_t)src[i]];
        for (size_t j = 0; j < d.pages.size(); j++) {
            if (d.pages[j] >= 0 && share) k->refs[(size_t)d.pages[j]]++;
            if (d.pages[j] >= 0 && !share) {
                pairs.emplace_back(d.pages[j], k->take());
                d.pages[j] = pairs.back().second;
            }
            ch.add((int64_t)dst[i] * k->c.sequence_pages + (int64_t)j, d.pages[j]);
        }
    }
    k->step_checked = false;
    c.order();
    copy_pages(c, pairs, false);
    ch.launch(c, true);
    return c.end_change("kv fork");
} catch (const std::exception &) {
    return no_memory("kv fork");
}

int j4q_kv_truncate(j4q_kv kv, const int32_t *seqs, const int64_t *lengths, int32_t n) try {
    std::lock_guard<std::mutex> lk(abi::lock());
    Kv *k;
    int rc = get(kv, "kv truncate", &k);
    if (rc) return rc;
    if (!lengths) return report_error(J4Q_EINVAL, "kv truncate: lengths is NULL");
    if ((rc = check_seqs(*k, "kv truncate", seqs, n, true))) return rc;
    const int64_t per = k->c.page_tokens;
    for (int32_t i = 0; i < n; i++) {
        const Seq &q = k->seqs[(size_t)seqs[i]];
        if (lengths[i] < 0 || lengths[i] > q.len)
            return report_error(J4Q_EINVAL, "kv truncate: sequence %d has %lld tokens, not %lld", seqs[i], (long long)q.len, (long long)lengths[i]);
        if (lengths[i] % per && q.pages[(size_t)(lengths[i] / per)] < 0)
            return report_error(J4Q_EINVAL, "kv truncate: sequence %d would end in an evicted page", seqs[i]);
    }
    for (int32_t i = 0; i < n; i++) {
        Seq &q = k->seqs[(size_t)seqs[i]];
        if (lengths[i] == q.len) continue;
        if (in_step(*k, seqs[i])) end_step(*k);
        q.len = lengths[i];
        while ((int64_t)q.pages.size() > (q.len + per - 1) / per) {
            k->drop(q.pages.back());
            q.pages.pop_back();
        }
        q.gone1 = std::min(q.gone1, q.len);
        if (q.gone0 >= q.gone1) q.gone0 = q.gone1 = 0;
    }
    return J4Q_OK;
} catch (const std::exception &) {
    return no_memory("kv truncate");
}

int j4q_kv_evict(j4q_kv kv, const int32_t *seqs, int32_t n, int32_t window, int32_t sinks, void *stream) try {
    std::lock_guard<std::mutex> lk(abi::lock());
    Kv *k;
    int rc = get(kv, "kv evict", &k);
    if (rc) return rc;
    if (window < 1 || sinks < 0) return report_error(J4Q_EINVAL, "kv evict: a window of %d tokens, %d first ones (at least 1, 0)", window, sinks);
    if ((rc = check_seqs(*k, "kv evict", seqs, n, true))) return rc;
    if ((rc = abi::ready_locked())) return rc;
    Call c(*k, stream);
    if ((rc = c.check("kv evict", kChanges))) return rc;
    const int64_t per = k->c.page_tokens, first = (sinks + per - 1) / per;
    // the next token, at place len, sees j > len - window and j < sinks; an earlier one sees more
    auto last = [&](const Seq &q) { return std::max<int64_t>(0, (q.len - window + 1) / per); };
    Changes ch;
    for (int32_t i = 0; i < n; i++) {
        const Seq &q = k->seqs[(size_t)seqs[i]];
        for (int64_t p = first, end = last(q); p < end; p++)
            if (q.pages[(size_t)p] >= 0) ch.add((int64_t)seqs[i] * k->c.sequence_pages + p, -1);
    }
    for (int32_t i = 0; i < n; i++) {
        Seq &q = k->seqs[(size_t)seqs[i]];
        const int64_t end = last(q);
        if (first >= end) continue;
        for (int64_t p = first; p < end; p++) {
            k->drop(q.pages[(size_t)p]);
            q.pages[(size_t)p] = -1;
        }
        q.gone0 = q.gone1 ? std::min(q.gone0, first * per) : first * per;
        q.gone1 = std::max(q.gone1, end * per);
    }
    k->step_checked = false;
    c.order();
    ch.launch(c, true);
    return c.end_change("kv evict");
} catch (const std::exception &) {
    return no_memory("kv evict");
}

int j4q_kv_compact(j4q_kv kv, int64_t *moved, void *stream) try {
    std::lock_guard<std::mutex> lk(abi::lock());
    Kv *k;
    int rc = get(kv, "kv compact", &k);
    if (rc) return rc;
    if ((rc = abi::ready_locked())) return rc;
    Call c(*k, stream);
    if ((rc = c.check("kv compact", kChanges))) return rc;
    const int64_t live = k->c.pages - k->free_pages;
    Pairs pairs;
    std::vector<int32_t> to((size_t)k->c.pages, -1);
    int64_t hole = 0;
    for (int64_t p = live; p < k->c.pages; p++) {
        if (!k->refs[(size_t)p]) continue;
        while (k->refs[(size_t)hole]) hole++;  // below `live`: as many holes there as pages behind
        pairs.emplace_back((int32_t)p, (int32_t)hole);
        to[(size_t)p] = (int32_t)hole;
        hole++;
    }
    Changes ch;
    if (!pairs.empty())
        for (int32_t s = 0; s < k->c.sequences; s++) {
            const Seq &q = k->seqs[(size_t)s];
            for (size_t j = 0; j < q.pages.size(); j++)
                if (q.pages[j] >= 0 && to[(size_t)q.pages[j]] >= 0) ch.add((int64_t)s * k->c.sequence_pages + (int64_t)j, to[(size_t)q.pages[j]]);
        }
    if (!pairs.empty())
        for (Seq &q : k->seqs)
            for (int32_t &p : q.pages)
                if (p >= 0 && to[(size_t)p] >= 0) p = to[(size_t)p];
    for (const auto &[p, h] : pairs) {
        k->refs[(size_t)h] = k->refs[(size_t)p];
        k->refs[(size_t)p] = 0;
        k->free_bits[(size_t)(h / 64)] &= ~(1ull << (h % 64));
        k->free_bits[(size_t)(p / 64)] |= 1ull << (p % 64);
    }
    k->hint = 0;
    while (k->hint + 1 < (int64_t)k->free_bits.size() && !k->free_bits[(size_t)k->hint]) k->hint++;
    if (moved) *moved = (int64_t)pairs.size();
    if (pairs.empty()) return J4Q_OK;
    c.order();
    copy_pages(c, pairs, false);
    ch.launch(c, true);
    return c.end_change("kv compact");
} catch (const std::exception &) {
    return no_memory("kv compact");
}

int j4q_kv_append(j4q_kv kv, int32_t layer, const j4q_kv_append_args *args, void *stream) try {
    if (!args) return report_error(J4Q_EINVAL, "kv append: args is NULL");
    std::lock_guard<std::mutex> lk(abi::lock());
    Kv *k;
    int rc = get(kv, "kv append", &k);
    if (rc) return rc;
    const j4q_kv_append_args &g = *args;
    if (layer < 0 || layer >= k->c.layers) return report_error(J4Q_EINVAL, "kv append: layer %d out of range [0, %d)", layer, k->c.layers);
    if (!g.k || !g.v) return report_error(J4Q_EINVAL, "kv append: NULL k or v");
    if (!dense_type(g.type)) return report_error(J4Q_EUNSUPPORTED, "kv append: type %d (J4Q_KIND_F32 or J4Q_KIND_BF16)", g.type);
    if (k->step_seq.empty()) return report_error(J4Q_EINVAL, "kv append: no step (j4q_kv_extend begins one)");
    KvAppend a;
    a.kv_stride = g.kv_stride;
    a.q_stride = g.q_stride;
    const int64_t width = (int64_t)k->c.kv_heads * k->c.head_dim;
    if ((rc = check_stride("kv append", "k", g.k, g.type, width, &a.kv_stride)) || (rc = check_stride("kv append", "v", g.v, g.type, width, &a.kv_stride)))
        return rc;
    a.heads = 0;
    if (g.q) {
        if (g.heads < 1 || g.heads > 65535 || !g.q_out) return report_error(J4Q_EINVAL, "kv append: q needs q_out and its heads, got %d", g.heads);
        const int64_t q_width = (int64_t)g.heads * k->c.head_dim;
        if ((rc = check_stride("kv append", "q", g.q, g.type, q_width, &a.q_stride)) ||
            (rc = check_stride("kv append", "q_out", g.q_out, g.type, q_width, &a.q_stride)))
            return rc;
        a.heads = g.heads;
    }
    const int64_t e = g.type == J4Q_KIND_BF16 ? 2 : 4, q_bytes = (int64_t)a.heads * k->c.head_dim * e;
    if (g.q && ((g.q != g.q_out && overlap(g.q, a.q_stride * e, q_bytes, g.q_out, a.q_stride * e, q_bytes, k->step_rows)) ||
                overlap(g.k, a.kv_stride * e, width * e, g.q_out, a.q_stride * e, q_bytes, k->step_rows) ||
                overlap(g.v, a.kv_stride * e, width * e, g.q_out, a.q_stride * e, q_bytes, k->step_rows)))
        return report_error(J4Q_EUNSUPPORTED, "kv append: q_out overlaps k, v, or q without being q itself");
    if ((rc = fill_rope("kv append", g.rope, k->c.head_dim, k->step_rows, false, &a.rope))) return rc;
    if (!k->step_checked) {
        for (size_t i = 0; i < k->step_seq.size(); i++) {
            const Seq &q = k->seqs[(size_t)k->step_seq[i]];
            for (int64_t p = (q.len - k->step_tokens[i]) / k->c.page_tokens; p < (int64_t)q.pages.size(); p++)
                if (q.pages[(size_t)p] < 0 || k->refs[(size_t)q.pages[(size_t)p]] > 1)
                    return report_error(J4Q_EINVAL, "kv append: sequence %d's page %lld is %s", k->step_seq[i], (long long)p,
                                        q.pages[(size_t)p] < 0 ? "evicted" : "shared (the sequence was forked behind its j4q_kv_extend)");
        }
        k->step_checked = true;
    }
    a.l = k->layer(layer);
    a.step = k->step();
    a.k = g.k;
    a.v = g.v;
    a.q = g.q;
    a.q_out = g.q_out;
    a.bf16 = g.type == J4Q_KIND_BF16;
    if ((rc = abi::ready_locked())) return rc;
    Call c(*k, stream);
    if ((rc = c.check("kv append", nullptr))) return rc;
    // workgroups by sequence, unless the steps are so uneven that most of them would have nothing to do
    int64_t most = k->step_most_blocks, blocks = k->step_blocks;
    if (c.captured) {  // a replay's tokens may lie across one block more
        most = blocks = 0;
        for (int32_t t : k->step_tokens) {
            const int64_t b = (t - 1 + kKvBlock - 1) / kKvBlock + 1;
            most = std::max(most, b);
            blocks += b;
        }
    }
    const int64_t even = most * (int64_t)k->step_seq.size();
    a.max_blocks = even <= 4 * blocks ? (int32_t)most : 0;
    const int64_t items = a.max_blocks ? even : blocks;
    if (items * k->c.kv_heads + (int64_t)k->step_rows * a.heads > INT_MAX)
        return report_error(J4Q_EUNSUPPORTED, "kv append: %d tokens of %d heads in a call", k->step_rows, std::max(a.heads, k->c.kv_heads));
    a.items = (int32_t)items;
    c.order();
    if (c.e == hipSuccess) c.e = launch_kv_append(a, c.s, c.event(true));
    return c.end("kv append");
} catch (const std::exception &) {
    return no_memory("kv append");
}

int j4q_kv_attend(j4q_kv kv, int32_t layer, const j4q_kv_attend_args *args, void *stream) try {
    if (!args) return report_error(J4Q_EINVAL, "kv attend: args is NULL");
    std::lock_guard<std::mutex> lk(abi::lock());
    Kv *k;
    int rc = get(kv, "kv attend", &k);
    if (rc) return rc;
    const j4q_kv_attend_args &g = *args;
    if (layer < 0 || layer >= k->c.layers) return report_error(J4Q_EINVAL, "kv attend: layer %d out of range [0, %d)", layer, k->c.layers);
    if (!g.q || !g.out) return report_error(J4Q_EINVAL, "kv attend: NULL q or out");
    if (!dense_type(g.q_type) || !dense_type(g.out_type))
        return report_error(J4Q_EUNSUPPORTED, "kv attend: types %d, %d (J4Q_KIND_F32 or J4Q_KIND_BF16)", g.q_type, g.out_type);
    if (g.heads < 1 || g.heads % k->c.kv_heads || g.heads > 65535)
        return report_error(J4Q_EINVAL, "kv attend: %d query heads over %d kv heads", g.heads, k->c.kv_heads);
    if (g.window < 0 || g.sinks < 0) return report_error(J4Q_EINVAL, "kv attend: a window of %d tokens, %d first ones", g.window, g.sinks);
    if (!(g.scale >= 0.0f) || g.scale > 1e30f) return report_error(J4Q_EINVAL, "kv attend: scale %g", (double)g.scale);
    if (k->step_seq.empty()) return report_error(J4Q_EINVAL, "kv attend: no step (j4q_kv_extend or j4q_kv_begin begin one)");
    KvAttend a;
    a.q_stride = g.q_stride;
    a.out_stride = g.out_stride;
    const int64_t width = (int64_t)g.heads * k->c.head_dim;
    if ((rc = check_stride("kv attend", "q", g.q, g.q_type, width, &a.q_stride)) ||
        (rc = check_stride("kv attend", "out", g.out, g.out_type, width, &a.out_stride)))
        return rc;
    const int64_t qe = g.q_type == J4Q_KIND_BF16 ? 2 : 4, oe = g.out_type == J4Q_KIND_BF16 ? 2 : 4;
    if ((g.q != g.out || g.q_type != g.out_type || a.q_stride != a.out_stride) &&
        overlap(g.q, a.q_stride * qe, width * qe, g.out, a.out_stride * oe, width * oe, k->step_rows))
        return report_error(J4Q_EUNSUPPORTED, "kv attend: out overlaps q without being q itself");
    a.window = g.window ? g.window : INT_MAX;
    a.sinks = g.sinks;
    a.group = g.heads / k->c.kv_heads;
    const int n = (int)k->step_seq.size();
    const int some_rows = k->c.head_dim <= 128 ? kSomeRows : kFewRows;
    int64_t few = 0, some = 0, many = 0;  // most rows of a sequence and kv head that each kernel has
    for (int i = 0; i < n; i++) {
        const Seq &q = k->seqs[(size_t)k->step_seq[(size_t)i]];
        const int64_t first = q.len - k->step_tokens[(size_t)i], rows = (int64_t)k->step_tokens[(size_t)i] * a.group;
        if (q.gone1 > q.gone0 && (q.gone1 - 1 > first - a.window || q.gone0 < a.sinks))
            return report_error(J4Q_EINVAL, "kv attend: tokens [%lld, %lld) of sequence %d are evicted, and the mask shows some of them",
                                (long long)q.gone0, (long long)q.gone1, k->step_seq[(size_t)i]);
        int64_t &most = rows > some_rows ? many : rows > kFewRows ? some : few;
        most = std::max(most, rows);
    }
    if (many > 1 << 22 || n > 65535)
        return report_error(J4Q_EUNSUPPORTED, "kv attend: %lld query rows of %d kv heads in %d sequences", (long long)std::max(few, many), k->c.kv_heads, n);
    a.l = k->layer(layer);
    a.step = k->step();
    a.q = g.q;
    a.out = g.out;
    a.q_bf16 = g.q_type == J4Q_KIND_BF16;
    a.out_bf16 = g.out_type == J4Q_KIND_BF16;
    a.scale = (g.scale > 0.0f ? g.scale : 1.0f / sqrtf((float)k->c.head_dim)) * 1.4426950408889634f;
    a.part = k->part;
    a.part_ml = k->part + kPartRows * k->c.head_dim;
    if ((rc = abi::ready_locked())) return rc;
    Call c(*k, stream);
    if ((rc = c.check("kv attend", nullptr))) return rc;
    c.order();
    // sequences of few rows, of some and of many, in a launch each
    if (few && c.e == hipSuccess) {
        a.rows_from = 1, a.rows_to = kFewRows, a.max_rows = (int32_t)few;
        split_few(*k, c.captured, &a);
        c.e = launch_kv_decode(a, c.s, c.event(!some && !many));
    }
    if (some && c.e == hipSuccess) {
        a.rows_from = kFewRows + 1, a.rows_to = some_rows, a.max_rows = (int32_t)some;
        split_some(*k, c.captured, &a);
        c.e = launch_kv_rows(a, c.s, c.event(!many));
    }
    if (many && c.e == hipSuccess) {
        a.rows_from = some_rows + 1, a.rows_to = INT_MAX, a.max_rows = (int32_t)many;
        split_many(*k, c.captured, &a);
        c.e = launch_kv_prefill(a, c.s, c.event(true));
    }
    return c.end("kv attend");
} catch (const std::exception &) {
    return no_memory("kv attend");
}

int j4q_kv_read(j4q_kv kv, int32_t layer, const int32_t *seqs, const int64_t *first, int64_t count, int32_t n, float *k_out, float *v_out, void *stream) try {
    std::lock_guard<std::mutex> lk(abi::lock());
    Kv *k;
    int rc = get(kv, "kv read", &k);
    if (rc) return rc;
    if (layer < 0 || layer >= k->c.layers) return report_error(J4Q_EINVAL, "kv read: layer %d out of range [0, %d)", layer, k->c.layers);
    if (!first || (!k_out && !v_out)) return report_error(J4Q_EINVAL, "kv read: NULL argument");
    if (!aligned(k_out, 16) || !aligned(v_out, 16)) return report_error(J4Q_EINVAL, "kv read: outputs must be 16-byte aligned");
    if ((rc = check_seqs(*k, "kv read", seqs, n, false))) return rc;
    if (count < 1 || count > 1 << 30 || (count / kKvBlock + 2) * k->c.kv_heads * std::min<int64_t>(n, kKvReadSeqs) > INT_MAX)
        return report_error(J4Q_EINVAL, "kv read: %lld tokens", (long long)count);
    for (int32_t i = 0; i < n; i++)
        if (first[i] < 0 || first[i] > 1 << 30) return report_error(J4Q_EINVAL, "kv read: first token %lld", (long long)first[i]);
    if ((rc = abi::ready_locked())) return rc;
    Call c(*k, stream);
    if ((rc = c.check("kv read", "lengths of now, which a captured graph would repeat"))) return rc;
    c.order();
    for (int32_t at = 0; at < n && c.e == hipSuccess; at += kKvReadSeqs) {
        KvRead r;
        r.l = k->layer(layer);
        r.table = k->words;
        r.sequence_pages = k->c.sequence_pages;
        r.n = std::min(n - at, kKvReadSeqs);
        r.count = count;
        const int64_t skip = (int64_t)at * count * k->c.kv_heads * k->c.head_dim;
        r.k = k_out ? k_out + skip : nullptr;
        r.v = v_out ? v_out + skip : nullptr;
        for (int i = 0; i < r.n; i++) {
            r.seq[i] = seqs[at + i];
            r.first[i] = (int32_t)first[at + i];
            r.len[i] = (int32_t)k->seqs[(size_t)seqs[at + i]].len;
        }
        c.e = launch_kv_read(r, c.s, c.event(at + kKvReadSeqs >= n));
    }
    return c.end("kv read");
} catch (const std::exception &) {
    return no_memory("kv read");
}

int j4q_rope_into(const void *x, void *out, int type, int64_t rows, int32_t heads, int32_t head_dim, int64_t x_stride, int64_t out_stride,
                  const j4q_rope *rope, void *stream) {
    if (!x || !out || !rope) return report_error(J4Q_EINVAL, "rope_into: NULL argument");
    if (!dense_type(type)) return report_error(J4Q_EUNSUPPORTED, "rope_into: type %d (J4Q_KIND_F32 or J4Q_KIND_BF16)", type);
    if (rows < 1 || rows > 1 << 30 || heads < 1 || heads > 65535 || head_dim < 2 || head_dim % 2 || head_dim > kRopeMaxDim)
        return report_error(J4Q_EINVAL, "rope_into: %lld rows of %d heads of %d (an even number up to 2048)", (long long)rows, heads, head_dim);
    const int64_t width = (int64_t)heads * head_dim;
    if (!x_stride) x_stride = width;
    if (!out_stride) out_stride = width;
    if (x_stride < width || out_stride < width || x_stride > 1ll << 40 || out_stride > 1ll << 40)
        return report_error(J4Q_EINVAL, "rope_into: rows less than %lld values apart", (long long)width);
    const uintptr_t e = type == J4Q_KIND_BF16 ? 2 : 4;
    if (!aligned(x, e) || !aligned(out, e)) return report_error(J4Q_EINVAL, "rope_into: x and out must be aligned to their values");
    if (rows > (INT64_MAX >> 20) / width)
        return report_error(J4Q_EUNSUPPORTED, "rope_into: %lld rows of %lld values", (long long)rows, (long long)width);
    const int64_t b = (int64_t)e;
    if ((x != out || x_stride != out_stride) && overlap(x, x_stride * b, width * b, out, out_stride * b, width * b, rows))
        return report_error(J4Q_EUNSUPPORTED, "rope_into: out overlaps x without being x itself");
    KvRope r;
    int rc = fill_rope("rope_into", rope, head_dim, rows, true, &r);
    if (rc) return rc;
    std::lock_guard<std::mutex> lk(abi::lock());
    if ((rc = abi::ready_locked())) return rc;
    const hipError_t err = launch_rope(x, out, rows, heads, head_dim, x_stride, out_stride, type == J4Q_KIND_BF16, r, stream ? (hipStream_t)stream : abi::stream());
    return err == hipSuccess ? J4Q_OK : report_hip("rope_into", err);
}

}  // extern "C"
