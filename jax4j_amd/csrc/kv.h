// The 8-bit key/value cache: its layout in memory and what its kernels are given. The host side (pages, tables, checks,
// entry points) is kv.hip; kernels are in kv_write.hip (rotary positions, append, read, copies of pages), kv_decode.hip
// (attention of few query rows) and kv_prefill.hip (of some, and of many).
//
// A pool holds [layer][page]; a page holds page_tokens (16, 32 or 64) consecutive tokens of one sequence in one layer:
//   [kv head][block of 16 tokens] { K: int8 [16][D] | V: int8 [D][16] }   then   [kv head][block] { float K scale, V scale }
// K is stored by token and V by channel, so that 16 bytes at either are an operand of the int8 matrix instructions
// (16 channels of a key; 16 tokens of a value channel) and no kernel transposes. A value is code * scale of its block and
// head. Codes that nothing was written to are any int8 and weigh nothing; scales of blocks behind the end of a sequence
// are not used.
#pragma once

#include "j4q_common.h"

namespace j4q {

constexpr int kKvBlock = 16;                 // tokens that share a scale
constexpr int kKvTile = 64;                  // tokens that the attention kernels take at a time
constexpr float kKvMinScale = 0x1p-64f;      // of a block of zeros; keeps 1 / scale and sums of weight / scale far inside fp32
constexpr int kKvMaxDim = 256;

__host__ __device__ inline int64_t kv_page_bytes(int kv_heads, int dim, int page_tokens) {
    const int64_t blocks = (int64_t)kv_heads * (page_tokens / kKvBlock);
    return (int64_t)align256((uint64_t)(blocks * (2 * kKvBlock * dim + 8)));
}

// One layer of a pool.
struct KvLayer {
    uint8_t *base;
    int64_t page_bytes;
    int32_t scales;       // byte offset of the scales in a page
    int32_t kv_heads, dim;
    int32_t block_shift;  // a page has 1 << block_shift blocks
};

// The current step: sequence seq[i] has len[i] tokens, of which the last row0[i + 1] - row0[i] are the step's, rows
// row0[i].. of the caller's q, k, v and out.
struct KvStep {
    const int32_t *table;  // [sequences][sequence_pages], -1: no page
    const int32_t *seq, *len, *row0;
    const int32_t *block0;  // [n + 1]: blocks of 16 that the step's tokens touch, of the sequences before
    int32_t sequence_pages;
    int32_t n, rows;       // sequences and rows of the step
};

// Rotary positions: pair i of a row is turned by cos/sin[position of axis[i]][i]. pairs == 0: none.
struct KvRope {
    const float *cos, *sin;    // [table_rows][pairs]
    const int32_t *positions;  // [axes][rows]; nullptr: a token's place in its sequence
    int32_t table_rows, pairs, axes;
    int32_t interleaved;       // pair i: channels 2i, 2i + 1; else i, i + pairs
    int32_t rows;              // row pitch of positions
    uint8_t axis[kKvMaxDim / 2];
};

struct KvAttend {
    KvLayer l;
    KvStep step;
    const void *q;
    void *out;
    int64_t q_stride, out_stride;  // elements from a row to the next
    int32_t q_bf16, out_bf16;
    int32_t group;                 // query heads of a kv head
    int32_t window, sinks;         // window: INT32_MAX for none
    float scale;                   // of the scores, times log2(e)
    int32_t row_tile;              // rows of a workgroup
    int32_t rows_from, rows_to;    // rows (tokens x group) of the sequences that the launch serves
    int32_t max_rows;              // most rows (tokens x group) of a sequence and kv head in the step
    int32_t splits;                // ranges of the visible tokens, one workgroup each
    int32_t split_tiles;           // tiles of a range (kv_range_tiles)
    float *part;                   // splits > 1: [sequence][kv head][row][split][D], then {max, sum} [...][split]
    float *part_ml;
};

// Tiles of 64 tokens that any of the rows at positions first.. of a sequence sees: [0, sink) and [low, end).
struct KvTiles {
    int sink, low, end;
    __host__ __device__ int count() const { return sink + end - low; }
    __host__ __device__ int tile(int i) const { return i < sink ? i : i - sink + low; }
};
__host__ __device__ inline KvTiles kv_tiles(int first, int last, int window, int sinks) {
    KvTiles t{0, 0, 0};
    if (last < 0) return t;
    const int low = first - window + 1 > 0 ? first - window + 1 : 0;
    t.end = last / kKvTile + 1;
    t.low = low / kKvTile;
    t.sink = (sinks < low ? sinks + kKvTile - 1 : low) / kKvTile;
    if (t.sink > t.low) t.sink = t.low;
    return t;
}
// Tiles of a range where a row's are `tiles`, and how many ranges these are (the last one takes what is left). A later run of a
// captured call may have more tiles than `splits` ranges of split_tiles hold: all its ranges grow then, or the last one would
// walk the rest alone (8 kv heads, 128 query heads, a step of 32 tokens captured at a length of 128 and run at 8192, into bf16:
// 15 ranges of 2 tiles and one of 98 took 216 us, 16 of 8 take 48).
__host__ __device__ inline int kv_range_tiles(int tiles, const KvAttend &a) {
    return tiles <= a.splits * a.split_tiles ? a.split_tiles : (tiles + a.splits - 1) / a.splits;
}
__host__ __device__ inline int kv_ranges(int tiles, const KvAttend &a) {
    const int each = kv_range_tiles(tiles, a);
    return (tiles + each - 1) / each;
}

constexpr int kKvSplits = 256;  // most ranges of a row's tokens
hipError_t launch_kv_decode(const KvAttend &a, hipStream_t s, hipEvent_t done);
hipError_t launch_kv_rows(const KvAttend &a, hipStream_t s, hipEvent_t done);
hipError_t launch_kv_prefill(const KvAttend &a, hipStream_t s, hipEvent_t done);
// The parts of every row in one: out = sum of part * 2^(max - largest) / the same of the sums.
hipError_t launch_kv_join(const KvAttend &a, hipStream_t s, hipEvent_t done);

struct KvAppend {
    KvLayer l;
    KvStep step;
    const void *k, *v, *q;
    void *q_out;
    int64_t kv_stride, q_stride;
    int32_t bf16, heads;  // heads: of q (0: no q)
    int32_t rows_each, heads_each, wide;  // of a workgroup that turns queries (the launcher's)
    int32_t max_blocks;   // workgroups (per kv head) for each sequence; 0: as many as it touches blocks (step.block0)
    int32_t items;        // ... of all sequences
    KvRope rope;
};
hipError_t launch_kv_append(const KvAppend &a, hipStream_t s, hipEvent_t done);
constexpr int kRopeMaxDim = 2048;
hipError_t launch_rope(const void *x, void *out, int64_t rows, int32_t heads, int32_t dim, int64_t stride, int64_t out_stride, bool bf16,
                       const KvRope &rope, hipStream_t s);

// Lists that kernels get in their arguments (of 4 KiB at most), in two sizes: the host writes all of a launch's
// arguments, whatever part of them is used (a read of 64 sequences: 4.5 us a call with the long list, 3.7 with the short).
constexpr int kKvReadSeqs = 256;
template <int N>
struct KvReadOf {
    KvLayer l;
    const int32_t *table;
    int32_t sequence_pages, n;
    int64_t count;
    float *k, *v;  // [n][count][kv heads][D]
    int32_t seq[N], first[N], len[N];
};
using KvRead = KvReadOf<kKvReadSeqs>;
hipError_t launch_kv_read(const KvRead &r, hipStream_t s, hipEvent_t done);

// words[at + j] = value + step * j, j < count.
struct KvRun {
    int32_t at, value, step, count;
};
constexpr int kKvRuns = 240;
template <int N>
struct KvRunsOf {
    int32_t *words;
    int32_t n;
    KvRun run[N];
};
using KvRuns = KvRunsOf<kKvRuns>;
hipError_t launch_kv_runs(const KvRuns &r, hipStream_t s, hipEvent_t done);

constexpr int kKvPairs = 480;
template <int N>
struct KvPairsOf {
    uint8_t *pool;
    int64_t page_bytes, layer_bytes;
    int32_t layers, n;
    int32_t src[N], dst[N];
};
using KvPairs = KvPairsOf<kKvPairs>;
hipError_t launch_kv_copy(const KvPairs &p, hipStream_t s, hipEvent_t done);

}  // namespace j4q
