// 16 rows of W as the matrix cores take them, exact codes (experts.h): unpacking, and products with a slice of x'.
//
// Codes are exact fp16 whole numbers with their offset (q - 8, q - 32, q), products of 32 (Q6_K: 16) with one scale come out of
// v_mfma_f32_16x16x32_f16 (16x16x16) in fp32 and are folded by one FMA with that scale; Q4_K's minima times the block's sums of x' by
// v_mfma_f32_16x16x4_f32.
#pragma once

#include "experts.h"

namespace j4q {
namespace ex {

__device__ __forceinline__ h2 as_h2(uint32_t v) { return __builtin_bit_cast(h2, v); }
__device__ __forceinline__ uint32_t bits(h2 v) { return __builtin_bit_cast(uint32_t, v); }
__device__ __forceinline__ h2 both(float v) { return h2{(_Float16)v, (_Float16)v}; }

// Half a slice of row n = lane % 16 of W as lane group g = lane / 16 uses it: dword g of each of 4 blocks of 16 bytes (Q8_0: of the
// two halves of each of 2 blocks) in v, Q6_K's high bits that belong to it in h.
template <int FMT>
struct Raw {
    uint32_t v[4], h[FMT == Q6_K ? 4 : 1];
    u32x4 s;     // of the whole slice. Q8_0, Q4_0: fp16 scales of the blocks; Q4_K: the superblock's header; Q6_K: 16 int8 scales
    uint32_t d;  // Q6_K: fp16 d
};

// The 8 codes of a dword (and Q6_K's high bits, or Q8_0's dword of the block's second half) as fp16 whole numbers.
// `one`: 1024 and 1024, below which the bits are whole numbers, in a register (or_one()): a mask and that are one v_and_or then.
__device__ __forceinline__ uint32_t or_one() {
    uint32_t one = 0x64006400u;
    asm("" : "+v"(one));
    return one;
}
template <int FMT>
__device__ __forceinline__ h8 codes(uint32_t v, uint32_t more, uint32_t one) {
    u32x4 r;
    if constexpr (FMT == Q8_0) {
        const uint32_t a = v ^ 0x80808080u, b = more ^ 0x80808080u;
        const h2 off = both(-1152.f);
        r[0] = bits(as_h2((a & 0x00FF00FFu) | one) + off);
        r[1] = bits(as_h2((a >> 8 & 0x00FF00FFu) | one) + off);
        r[2] = bits(as_h2((b & 0x00FF00FFu) | one) + off);
        r[3] = bits(as_h2((b >> 8 & 0x00FF00FFu) | one) + off);
    } else {
        constexpr float o = FMT == Q4_0 ? 8.f : FMT == Q6_K ? 32.f : 0.f;
        const uint32_t t = v >> 8;
        uint32_t e0 = (v & 0x000F000Fu) | one, e1 = (t & 0x000F000Fu) | one, f0 = (v & 0x00F000F0u) | one, f1 = (t & 0x00F000F0u) | one;
        if constexpr (FMT == Q6_K) {
            const uint32_t u = more >> 2;
            asm("" : "+v"(e0), "+v"(e1), "+v"(f0), "+v"(f1));  // a second v_and_or each, not two masks and an or of three
            e0 = (more & 0x00300030u) | e0;
            e1 = (u & 0x00300030u) | e1;
            f0 = (more & 0x03000300u) | f0;
            f1 = (u & 0x03000300u) | f1;
        }
        const h2 low = both(-1024.f - o), sixteenth = both(0.0625f), high = both(-64.f - o);
        r[0] = bits(as_h2(e0) + low);
        r[1] = bits(as_h2(e1) + low);
        r[2] = bits(__builtin_elementwise_fma(as_h2(f0), sixteenth, high));  // exact: a whole number below 2^10
        r[3] = bits(__builtin_elementwise_fma(as_h2(f1), sixteenth, high));
    }
    return __builtin_bit_cast(h8, r);
}

// Half a slice of x', operand b of block b (Q8_0: two of them). Row m of an operand is a pair's x' (bf16), or with 8 pairs a tile their
// hi parts (m < 8) and lo parts (m >= 8), whose products come out in rows of their own.
template <int FMT>
struct Operands {
    h8 x[FMT == Q8_0 ? 2 : 4];
};

// Lane (m, g): the sum of row m in block g.
__device__ __forceinline__ float block_sum(const Operands<Q4_K> &a, int g) {
    h8 one;
#pragma unroll
    for (int j = 0; j < 8; j++) one[j] = (_Float16)1.f;
    float s[4];
#pragma unroll
    for (int t = 0; t < 4; t++) s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(one, a.x[t], f32x4{}, 0, 0, 0)[0];
    return g < 2 ? (g ? s[1] : s[0]) : (g == 2 ? s[2] : s[3]);
}

// acc - low += x' . W tile over half i of a slice (low: Q4_K's minima); lane (n, g): rows 4 g + j of the operand, row n of W.
template <int FMT>
__device__ __forceinline__ void multiply(const Raw<FMT> &r, const Operands<FMT> &a, int i, int g, uint32_t one, f32x4 &acc, f32x4 &low) {
    if constexpr (FMT == Q8_0) {
#pragma unroll
        for (int t = 0; t < 2; t++) {
            const f32x4 c = __builtin_amdgcn_mfma_f32_16x16x32_f16(a.x[t], codes<FMT>(r.v[2 * t], r.v[2 * t + 1], one), f32x4{}, 0, 0, 0);
            const float d = (float)as_h2(r.s[i])[t];
#pragma unroll
            for (int j = 0; j < 4; j++) acc[j] = __builtin_fmaf(d, c[j], acc[j]);
        }
        return;
    }
    float scale[4];
    f32x4 part;  // Q6_K: before the superblock's scale
    if constexpr (FMT == Q4_K) {
        // lane group g decodes block 4 i + g
        const int sj = 4 * i + g;
        const uint32_t sc = __builtin_amdgcn_ubfe(r.s[1], 4 * sj, 4) | (__builtin_amdgcn_ubfe(r.s[3], 2 * sj, 2) << 4);
        const uint32_t mn = __builtin_amdgcn_ubfe(r.s[2], 4 * sj, 4) | (__builtin_amdgcn_ubfe(r.s[3], 16 + 2 * sj, 2) << 4);
        gmf::bcast4(half_bits_to_float(r.s[0] & 0xFFFFu) * (float)sc, scale);
        low = __builtin_amdgcn_mfma_f32_16x16x4f32(block_sum(a, g), half_bits_to_float(r.s[0] >> 16) * (float)mn, low, 0, 0, 0);
    } else if constexpr (FMT == Q4_0) {
#pragma unroll
        for (int t = 0; t < 4; t++) scale[t] = (float)as_h2(r.s[2 * i + t / 2])[t & 1];
    }
    // the products first: a fold waits for its own
    f32x4 c[4], c1[4];
#pragma unroll
    for (int t = 0; t < 4; t++) {
        if constexpr (FMT == Q6_K) {
            const h8 w = codes<FMT>(r.v[t], r.h[t], one);
            c[t] = __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_shufflevector(a.x[t], a.x[t], 0, 1, 2, 3), __builtin_shufflevector(w, w, 0, 1, 2, 3),
                                                         f32x4{}, 0, 0, 0);
            c1[t] = __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_shufflevector(a.x[t], a.x[t], 4, 5, 6, 7), __builtin_shufflevector(w, w, 4, 5, 6, 7),
                                                          f32x4{}, 0, 0, 0);
        } else {
            c[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a.x[t], codes<FMT>(r.v[t], 0u, one), f32x4{}, 0, 0, 0);
        }
    }
#pragma unroll
    for (int t = 0; t < 4; t++) {
        if constexpr (FMT == Q6_K) {
            const uint32_t sw = r.s[2 * i + t / 2] >> (16 * (t & 1));
            const float s0 = (float)(int8_t)(sw & 0xFFu), s1 = (float)(int8_t)(sw >> 8 & 0xFFu);
#pragma unroll
            for (int j = 0; j < 4; j++) part[j] = __builtin_fmaf(s1, c1[t][j], t ? __builtin_fmaf(s0, c[t][j], part[j]) : s0 * c[t][j]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++) acc[j] = __builtin_fmaf(scale[t], c[t][j], acc[j]);
        }
    }
    if constexpr (FMT == Q6_K) {
        const float d = half_bits_to_float(r.d);
#pragma unroll
        for (int j = 0; j < 4; j++) acc[j] = __builtin_fmaf(d, part[j], acc[j]);
    }
}

}  // namespace ex
}  // namespace j4q
