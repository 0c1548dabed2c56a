// The experts' products of a layer (j4q_experts_apply): out_r = sum_s w_rs down_e (act(gate_e x_r) * (up_e x_r)), e = ids_rs.
// Engine-local; the reference has no experts. What the kernels share; launches and checks: experts.hip.
//
// Pairs (row, slot) are put in the order of their experts, each expert's in the order of the rows, and cut into tiles of pairs that
// share an expert; all of it on the GPU, so that a call waits for nothing and may be captured. A launch per step:
//  1. experts_plan: order and tiles; x as fp16.   2. gate|up of every tile, the activation in its epilogue.
//  3. down of every tile, a weighted partial result for each pair.   4. experts_combine: the sums of a row's pairs, slot by slot.
//
// Activations enter the matrix cores as fp16: x' = x 2^e, e a power for each row that brings its largest magnitude into
// [2^14, 2^15), as one value (bf16 x: exact down to 2^-28 of the largest) or as hi + lo 2^-11 (fp32 x: 22 bits down to 2^-28; lo lies
// beside hi in size, and so in fp16's range where hi does). The inner activations are stored the same way, at a power that is known before
// they are: |g u| <= |x|^2 max(G U), with G and U the norms of a gate row and of the same up row, so h' = h 2^(14 - ceil(log2 of that))
// cannot overflow. Where the vectors are no worse than random the bound is about `dim` times what is typical: 2^12 of fp16's 2^29
// normal binades at dim 4096, which leaves 2^16 for rows larger than the others: 256 times in gate and up at once. (With lo at hi's
// own power, 22 bits ended 2^5 below what is typical: with such rows 32 times the others fp32 lost 5 bits, 256 times 11.)
//
// bf16 results of many pairs: a pair's partial result is fp16 on its way to a row's sum (11 bits before a rounding to 8), 64 columns at a
// power that takes the largest of them into [2^13, 2^14), known once they are computed, so that 11 bits reach down to 2^-28 of it whatever
// the sizes of the weights' rows. (At a power from bounds, as h' has it, one row of gate, up and down 32 times the others left up
// to 7 % of error in all other columns.) Half of fp32's bytes: 32744 pairs of dim 2048, 643 -> 574 us of the whole; the powers take 5 of them.
//
// Layout of x' and h' (block layout): of every 32 values, 16-byte chunk g = 0..3 holds elements 4 g + {0, 2, 1, 3} and then
// 16 + 4 g + {0, 2, 1, 3}: what masking dword g of a block of codes yields, for every type alike, so that a lane of the matrix core reads
// its 8 values with one load and codes are never reordered.
#pragma once

#include "gemv_lanes.h"
#include "j4q_common.h"

namespace j4q {
namespace ex {

using gmf::h2;
using gmf::h4;
using gmf::h8;
using gemv::Chunk;
using gemv::f32x4;
using gemv::kOob;
using gemv::make_rsrc;
using gemv::Offs;
using gemv::Rsrc;
using gemv::u32x2;
using gemv::u32x4;

constexpr int kBound = 14;       // |h'| <= 2^kBound
constexpr int kNothing = -4096;  // exponent of a norm of 0
constexpr float kLow = 2048.f;   // lo times this is stored

// A tile: pairs [first, first + count) of the order, all of one expert.
struct Tile {
    int32_t expert, first, count, pad;
};

// The tiles of gate|up's launch, or of down's.
struct Tiles {
    int rows;  // pairs of a tile
    int most;  // of the grid: no call has more
    int32_t *count;
    Tile *tile;
};

struct Weights {
    QMat gate, up, down;
    int up_type, down_type;
    int experts, dim, ffn, act;
    const int32_t *bound;                       // ceil(log2(max(G U))) of each expert
    const int32_t *gate_pow, *up_pow, *down_pow;  // of each row: max |w| 2^pow in [2^13, 2^14)
};

struct Call {
    const void *x;
    int64_t x_stride;  // values
    const int32_t *ids;
    const float *weights;
    void *out;
    int64_t out_stride;
    int rows, top, pairs;
    uint32_t top_inverse;  // ceil(2^32 / top); not used for 1
    bool half;      // bf16 x and out; x' and h' have no lo part
    bool one;       // a row, or very few, on their own kernels
    bool few;       // tiles of up to 16 pairs
    int splits;     // of down's K, whose partial results are added too
    Tiles up, down;
    // workspace
    int32_t *order;
    _Float16 *xa, *ha;         // hi; lo 2^11 behind all of hi
    int32_t *x_pow, *x_norm;   // of each row: e, and an exponent with |x| <= 2^it
    float *part;               // [splits][pairs][dim], times the weights; `small`: fp16 [pairs][dim] at powers part_pow, without them
    int32_t *part_pow;         // [pairs][dim / 64]: `small`: of each 64 columns of a pair
    bool small;
};

__device__ __forceinline__ int h_pow(const Weights &w, int expert, int x_norm) { return kBound - (2 * x_norm + w.bound[expert]); }

// pair / top: the inverse is above by less than top / 2^32 of itself, and pair * top < 2^32.
__device__ __forceinline__ int row_of(const Call &c, int pair) { return c.top == 1 ? pair : (int)__umulhi((uint32_t)pair, c.top_inverse); }

// Where element c of a row lies in the block layout.
__device__ __forceinline__ int slot_of(int c) {
    const int r = c & 15, i = r & 3;
    return (c & ~31) + 8 * (r >> 2) + 4 * (c >> 4 & 1) + ((i & 1) << 1 | i >> 1);
}

// e^x, within 3 steps: v_exp_f32 of the product with log2 e, and what the product's rounding left.
__device__ __forceinline__ float exp_of(float x) {
    constexpr float kLog2e = 1.44269504f, kRest = 1.92596303e-8f, kLn2 = 0.693147181f;
    const float t = x * kLog2e, e = __builtin_amdgcn_exp2f(t), rest = __builtin_fmaf(x, kRest, __builtin_fmaf(x, kLog2e, -t));
    return fabsf(t) < 128.f ? __builtin_fmaf(e, rest * kLn2, e) : e;
}

// v_rcp_f32 is within a step; where it is 0 (g below -88) so is the result.
__device__ __forceinline__ float activate(float g, int act) {
    if (act == 2) return g < 0.f ? 0.f : g;  // NaN stays NaN
    if (act == 1) {
        const float t = 0.7978845608028654f * (g + 0.044715f * g * g * g);
        return g * __builtin_amdgcn_rcpf(1.f + exp_of(-2.f * t));  // (1 + tanh t) / 2 = 1 / (1 + e^-2t)
    }
    return g * __builtin_amdgcn_rcpf(1.f + exp_of(-g));
}

// View of one expert's rows.
__device__ __forceinline__ QMat expert_of(const QMat &m, int fmt, int e, int64_t rows) {
    QMat o = m;
    const int64_t first = (int64_t)e * rows, k = m.cols;
    o.rows = rows;
    switch (fmt) {
    case Q8_0: o.qs += first * k; o.sc += first * (k / 16); break;
    case Q4_0:
    case Q4_K: o.qs += first * (k / 2); o.sc += first * (k / 16); break;
    default:
        o.qs += first * (k / 2);
        o.qh += first * (k / 4);
        o.sc += first * (k / 16);
        o.d += first * (k / 128);
        break;
    }
    return o;
}

// Rows of W as whole waves read them, a lane the 32 columns of a chunk.
// Byte offsets of chunk c of a row.
template <int FMT>
__device__ __forceinline__ Offs chunk_at(uint32_t c) {
    switch (FMT) {
    case Q4_0: return {16 * c, 0, 2 * c, 0};
    case Q8_0: return {32 * c, 0, 2 * c, 0};
    case Q4_K: return {16 * c, 0, (c >> 3) * 16, 0};
    default: return {16 * c, 8 * c, 2 * c, (c >> 3) * 2};
    }
}
// ... of a row of K columns.
template <int FMT>
__device__ __forceinline__ Offs row_bytes(uint32_t K) {
    switch (FMT) {
    case Q8_0: return {K, 0, K / 16, 0};
    case Q6_K: return {K / 2, K / 4, K / 16, K / 128};
    default: return {K / 2, 0, K / 16, 0};
    }
}

// The products of every tile: of up to 16 pairs (fp32: 8), or of rows_many(), by the type of the matrix.
int rows_many(int type, bool half, int each);
int splits_few(const Weights &w, int tiles);
hipError_t launch_few(const Weights &w, const Call &c, bool down, hipStream_t s);
hipError_t launch_many(const Weights &w, const Call &c, bool down, hipStream_t s);
// All of a call of very few rows, whose c.part is [pairs][ffn]; `done` as launch_with_event takes it.
bool one_fits(const Weights &w, int top);
hipError_t launch_one(const Weights &w, const Call &c, hipEvent_t done, hipStream_t s);

}  // namespace ex
}  // namespace j4q
