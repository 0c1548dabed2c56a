// Products of tiles of up to 16 pairs with an expert's rows, exact codes (experts.h).
//
// A workgroup has one tile of pairs and NT tiles of 16 rows of W (gate and up of the same columns, or down). K is split over its
// waves in slices of 256 columns: a wave turns its slice of x' into matrix-core operands once, which stay in registers for all NT
// tiles, and the loads of all NT tiles are in flight before the first is used; longer K comes round by round, each tile's registers
// refilled as soon as it has been used. The waves' sums meet in LDS, added in wave order.
//
// Codes are exact fp16 whole numbers with their offset (q - 8, q - 32, q), products of 32 (Q6_K: 16) with one scale come out of
// v_mfma_f32_16x16x32_f16 (16x16x16) in fp32 and are folded by one FMA with that scale; Q4_K's minima times the block's
// sums of x' by v_mfma_f32_16x16x4_f32. lo goes first: the matrix core aligns the products of one instruction and its C input to the
// largest, and drops what lies below.
#include "experts.h"

namespace j4q {
namespace ex {
namespace {

using gmf::bcast4;
using gmf::lane_off;
using gmf::ld128;
using gmf::ld16;
using gmf::ld64;
using gmf::xpose4;

__device__ __forceinline__ h2 as_h2(uint32_t v) { return __builtin_bit_cast(h2, v); }
__device__ __forceinline__ uint32_t bits(h2 v) { return __builtin_bit_cast(uint32_t, v); }
__device__ __forceinline__ h2 both(float v) { return h2{(_Float16)v, (_Float16)v}; }

// 16 rows x 256 columns of W as they are loaded: lane (n, g) = (lane % 16, lane / 16) has 16-byte units g, g + 4, ... of row n's codes.
template <int FMT>
struct Raw {
    u32x4 q[FMT == Q8_0 ? 4 : 2];
    u32x2 h[FMT == Q6_K ? 2 : 1];
    u32x4 s;     // Q8_0, Q4_0: 8 fp16 scales; Q4_K: the superblock's header; Q6_K: 16 int8 scales
    uint32_t d;  // Q6_K: fp16 d
};

template <int FMT>
struct Rows {
    __amdgpu_buffer_rsrc_t qs, qh, sc, d;
    __device__ __forceinline__ void init(const QMat &m) {
        const uint64_t rows = (uint64_t)m.rows, k = (uint64_t)m.cols;
        qs = make_rsrc(m.qs, rows * (FMT == Q8_0 ? k : k / 2));
        sc = make_rsrc(m.sc, rows * (k / 16));
        if constexpr (FMT == Q6_K) {
            qh = make_rsrc(m.qh, rows * (k / 4));
            d = make_rsrc(m.d, rows * (k / 128));
        }
    }
    // Slice sl (blocks 8 sl .. + 7) of row `row`; zeros where not ok and behind the row's last block.
    __device__ __forceinline__ void load(Raw<FMT> &r, uint32_t row, uint32_t K, uint32_t g, int sl, bool ok) const {
        const int left = (int)(K / 32) - 8 * sl;  // blocks from the slice's first on
        if constexpr (FMT == Q8_0) {
#pragma unroll
            for (int i = 0; i < 4; i++) r.q[i] = ld128(qs, row * K + 16u * g, (uint32_t)sl * 256u + 64u * i, ok && 2 * i < left);
        } else {
#pragma unroll
            for (int i = 0; i < 2; i++) r.q[i] = ld128(qs, row * (K / 2) + 16u * g, (uint32_t)sl * 128u + 64u * i, ok && 4 * i < left);
        }
        if constexpr (FMT == Q8_0 || FMT == Q4_0) {
            // rows of scales are 4- (Q8_0) or 8-byte aligned
#pragma unroll
            for (int i = 0; i < 4; i++)
                r.s[i] = gmf::ld32(sc, row * (K / 16) + 4u * i, (uint32_t)sl * 16u, ok && 2 * i < left);
        } else {
            r.s = ld128(sc, row * (K / 16), (uint32_t)sl * 16u, ok);
        }
        if constexpr (FMT == Q6_K) {
#pragma unroll
            for (int i = 0; i < 2; i++) r.h[i] = ld64(qh, row * (K / 4) + 8u * g, (uint32_t)sl * 64u + 32u * i, ok);
            r.d = ld16(d, row * (K / 128), (uint32_t)sl * 2u, ok);
        }
    }
};

// The 8 codes of a dword (and Q6_K's high bits, or Q8_0's dword of the block's second half) as fp16 whole numbers.
template <int FMT>
__device__ __forceinline__ h8 codes(uint32_t v, uint32_t more) {
    constexpr uint32_t one = 0x64006400u;  // 1024: the bits below are whole numbers
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
            e0 |= more & 0x00300030u;
            e1 |= u & 0x00300030u;
            f0 |= more & 0x03000300u;
            f1 |= u & 0x03000300u;
        }
        const h2 low = both(-1024.f - o), sixteenth = both(0.0625f), high = both(-64.f - o);
        r[0] = bits(as_h2(e0) + low);
        r[1] = bits(as_h2(e1) + low);
        r[2] = bits(__builtin_elementwise_fma(as_h2(f0), sixteenth, high));  // exact: a whole number below 2^10
        r[3] = bits(__builtin_elementwise_fma(as_h2(f1), sixteenth, high));
    }
    return __builtin_bit_cast(h8, r);
}

// A wave's slice of x': operand b of block b.
template <bool HL>
struct Operands {
    h8 hi[8], lo[HL ? 8 : 1];
    float sum[2];  // Q4_K: lane (m, g): the sum of x' of row m in blocks g and 4 + g
};

template <int FMT, bool HL>
__device__ __forceinline__ void block_sums(Operands<HL> &a, int g) {
    if constexpr (FMT == Q4_K) {
        h8 one;
#pragma unroll
        for (int j = 0; j < 8; j++) one[j] = (_Float16)1.f;
#pragma unroll
        for (int i = 0; i < 2; i++) {
            float s[4];
#pragma unroll
            for (int t = 0; t < 4; t++) {
                f32x4 c = {};
                if constexpr (HL) c = __builtin_amdgcn_mfma_f32_16x16x32_f16(one, a.lo[4 * i + t], c, 0, 0, 0);
                s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(one, a.hi[4 * i + t], c, 0, 0, 0)[0];
            }
            a.sum[i] = g < 2 ? (g ? s[1] : s[0]) : (g == 2 ? s[2] : s[3]);
        }
    }
}

template <int FMT, bool HL>
__device__ __forceinline__ f32x4 product(const Operands<HL> &a, int b, h8 w) {
    f32x4 c = {};
    if constexpr (HL) c = __builtin_amdgcn_mfma_f32_16x16x32_f16(a.lo[b], w, c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a.hi[b], w, c, 0, 0, 0);
}

// acc += x' slice . W tile; lane (n, g): rows 4 g + j of the pairs, row n of W.
template <int FMT, bool HL>
__device__ __forceinline__ void multiply(const Raw<FMT> &r, const Operands<HL> &a, int g, f32x4 &acc) {
    if constexpr (FMT == Q8_0) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            uint32_t v[4] = {r.q[i].x, r.q[i].y, r.q[i].z, r.q[i].w};
            xpose4(v);
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const f32x4 c = product<FMT, HL>(a, 2 * i + t, codes<FMT>(v[2 * t], v[2 * t + 1]));
                const float d = (float)as_h2(r.s[i])[t];
#pragma unroll
                for (int j = 0; j < 4; j++) acc[j] = __builtin_fmaf(d, c[j], acc[j]);
            }
        }
    } else {
        f32x4 low = {};
#pragma unroll
        for (int i = 0; i < 2; i++) {
            uint32_t v[4] = {r.q[i].x, r.q[i].y, r.q[i].z, r.q[i].w};
            xpose4(v);
            float scale[4];
            uint32_t high[4] = {};
            float d = 0.f;
            if constexpr (FMT == Q4_K) {
                // lane group g decodes block 4 i + g
                const int sj = 4 * i + g;
                const uint32_t sc = __builtin_amdgcn_ubfe(r.s[1], 4 * sj, 4) | (__builtin_amdgcn_ubfe(r.s[3], 2 * sj, 2) << 4);
                const uint32_t mn = __builtin_amdgcn_ubfe(r.s[2], 4 * sj, 4) | (__builtin_amdgcn_ubfe(r.s[3], 16 + 2 * sj, 2) << 4);
                bcast4(half_bits_to_float(r.s[0] & 0xFFFFu) * (float)sc, scale);
                low = __builtin_amdgcn_mfma_f32_16x16x4f32(a.sum[i], half_bits_to_float(r.s[0] >> 16) * (float)mn, low, 0, 0, 0);
            } else if constexpr (FMT == Q4_0) {
#pragma unroll
                for (int t = 0; t < 4; t++) scale[t] = (float)as_h2(r.s[2 * i + t / 2])[t & 1];
            } else {
                // lane group g holds dwords 0, 1 of block 4 i + g; block t needs dword g / 2, rotated right by 8 where g is odd
                const auto hs = __builtin_amdgcn_permlane32_swap(r.h[i].x, r.h[i].y, false, false);
                const auto e0 = __builtin_amdgcn_permlane16_swap(hs[0], hs[0], false, false);
                const auto e1 = __builtin_amdgcn_permlane16_swap(hs[1], hs[1], false, false);
                const uint32_t hq[4] = {e0[0], e0[1], e1[0], e1[1]};
#pragma unroll
                for (int t = 0; t < 4; t++) high[t] = __builtin_amdgcn_alignbit(hq[t], hq[t], (uint32_t)(g & 1) * 8u);
                d = half_bits_to_float(r.d);
            }
#pragma unroll
            for (int t = 0; t < 4; t++) {
                const int b = 4 * i + t;
                const h8 w = codes<FMT>(v[t], high[t]);
                if constexpr (FMT == Q6_K) {
                    f32x4 c0 = {}, c1 = {};
                    const h4 w0 = __builtin_shufflevector(w, w, 0, 1, 2, 3), w1 = __builtin_shufflevector(w, w, 4, 5, 6, 7);
                    if constexpr (HL) {
                        c0 = __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_shufflevector(a.lo[b], a.lo[b], 0, 1, 2, 3), w0, c0, 0, 0, 0);
                        c1 = __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_shufflevector(a.lo[b], a.lo[b], 4, 5, 6, 7), w1, c1, 0, 0, 0);
                    }
                    c0 = __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_shufflevector(a.hi[b], a.hi[b], 0, 1, 2, 3), w0, c0, 0, 0, 0);
                    c1 = __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_shufflevector(a.hi[b], a.hi[b], 4, 5, 6, 7), w1, c1, 0, 0, 0);
                    const uint32_t sw = r.s[b / 2] >> (16 * (b & 1));
                    const float s0 = d * (float)(int8_t)(sw & 0xFFu), s1 = d * (float)(int8_t)(sw >> 8 & 0xFFu);
#pragma unroll
                    for (int j = 0; j < 4; j++) acc[j] = __builtin_fmaf(s1, c1[j], __builtin_fmaf(s0, c0[j], acc[j]));
                } else {
                    const f32x4 c = product<FMT, HL>(a, b, w);
#pragma unroll
                    for (int j = 0; j < 4; j++) acc[j] = __builtin_fmaf(scale[t], c[j], acc[j]);
                }
            }
        }
        if constexpr (FMT == Q4_K) acc -= low;
    }
}

// grid: (ceil(N / (16 NT')), tiles over y and z), NT' = NT for down, NT / 2 for gate|up.
template <int FMT, bool HL, int WAVES, int NT, bool DOWN>
__global__ void __launch_bounds__(WAVES * 64)
experts_few(Weights w, Call c) {
    constexpr int COLS = DOWN ? NT : NT / 2;  // tiles of 16 columns of the result
    __shared__ float red[WAVES][NT][256];
    const int at = (int)(blockIdx.z * gridDim.y + blockIdx.y);
    if (at >= c.tile_count[0]) return;
    const Tile tile = c.tile[at];
    const int expert = __builtin_amdgcn_readfirstlane(tile.expert), count = __builtin_amdgcn_readfirstlane(tile.count),
              first = __builtin_amdgcn_readfirstlane(tile.first);
    const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int n = lane & 15, g = lane >> 4;
    const int K = DOWN ? w.ffn : w.dim, N = DOWN ? w.dim : w.ffn, slices = (K + 255) / 256;
    const int col0 = (int)blockIdx.x * COLS;  // first tile of 16 columns
    Rows<FMT> one, two;
    if constexpr (DOWN) {
        one.init(expert_of(w.down, FMT, expert, N));
    } else {
        one.init(expert_of(w.gate, FMT, expert, N));
        two.init(expert_of(w.up, FMT, expert, N));
    }
    // tile nt: down: columns 16 (col0 + nt); gate|up: of gate (even) and up (odd) 16 (col0 + nt / 2)
    auto load = [&](Raw<FMT> &r, int nt, int sl) __attribute__((always_inline)) {
        const int t = col0 + (DOWN ? nt : nt / 2);
        (DOWN || nt % 2 == 0 ? one : two).load(r, (uint32_t)(16 * t + n), (uint32_t)K, (uint32_t)g, sl, sl < slices && 16 * t < N);
    };
    Raw<FMT> raw[NT];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) load(raw[nt], nt, wave);
    // this lane's row of x' (pair n of the tile)
    const int64_t lo = DOWN ? (int64_t)c.pairs * w.ffn : (int64_t)c.rows * w.dim;
    const _Float16 *row = DOWN ? c.ha : c.xa;
    if (n < count) row += (int64_t)(DOWN ? first + n : c.order[first + n] / c.top) * K;
    f32x4 acc[NT] = {};
    for (int sl = wave; sl < slices; sl += WAVES) {
        Operands<HL> a;
#pragma unroll
        for (int b = 0; b < 8; b++) {
            const bool ok = n < count && 8 * sl + b < K / 32;
            a.hi[b] = h8{};
            if (ok) a.hi[b] = *reinterpret_cast<const h8 *>(row + (8 * sl + b) * 32 + 8 * g);
            if constexpr (HL) {
                a.lo[b] = h8{};
                if (ok) a.lo[b] = *reinterpret_cast<const h8 *>(row + lo + (8 * sl + b) * 32 + 8 * g);
            }
        }
        block_sums<FMT, HL>(a, g);
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            multiply<FMT, HL>(raw[nt], a, g, acc[nt]);
            load(raw[nt], nt, sl + WAVES);
        }
    }
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int j = 0; j < 4; j++) red[wave][nt][(4 * g + j) * 16 + n] = acc[nt][j];
    __syncthreads();
    for (int o = (int)threadIdx.x; o < COLS * 256; o += WAVES * 64) {
        const int ct = o >> 8, m = o >> 4 & 15, col = 16 * (col0 + ct) + (o & 15);
        if (m >= count || col >= N) continue;
        const int pair = c.order[first + m], token = pair / c.top, pow = h_pow(w, expert, c.x_norm[token]);
        if constexpr (DOWN) {
            float s = 0.f;
#pragma unroll
            for (int v = 0; v < WAVES; v++) s += red[v][ct][o & 255];
            c.part[(int64_t)pair * N + col] = __builtin_ldexpf(s * c.weights[pair], -pow);  // the weight first: the product alone may not fit
        } else {
            float a = 0.f, b = 0.f;
#pragma unroll
            for (int v = 0; v < WAVES; v++) {
                a += red[v][2 * ct][o & 255];
                b += red[v][2 * ct + 1][o & 255];
            }
            const int e = -c.x_pow[token];
            const float h = __builtin_ldexpf(activate(__builtin_ldexpf(a, e), w.act) * __builtin_ldexpf(b, e), pow);
            const _Float16 hi = (_Float16)h;
            _Float16 *const at = c.ha + (int64_t)(first + m) * w.ffn + slot_of(col);
            *at = hi;
            if constexpr (HL) at[(int64_t)c.pairs * w.ffn] = (_Float16)(h - (float)hi);
        }
    }
}

template <int FMT, bool HL, bool DOWN>
hipError_t launch(const Weights &w, const Call &c, hipStream_t s) {
    constexpr int NT = 4;
    const int K = DOWN ? w.ffn : w.dim, N = DOWN ? w.dim : w.ffn, cols = 16 * (DOWN ? NT : NT / 2);
    const int y = c.tiles < 32768 ? c.tiles : 32768;
    const dim3 grid((unsigned)((N + cols - 1) / cols), (unsigned)y, (unsigned)((c.tiles + y - 1) / y));
    if (K <= 1024) experts_few<FMT, HL, 4, NT, DOWN><<<grid, 256, 0, s>>>(w, c);
    else experts_few<FMT, HL, 8, NT, DOWN><<<grid, 512, 0, s>>>(w, c);
    return hipGetLastError();
}

template <int FMT>
hipError_t launch_type(const Weights &w, const Call &c, bool down, hipStream_t s) {
    if (down) return c.half ? launch<FMT, false, true>(w, c, s) : launch<FMT, true, true>(w, c, s);
    return c.half ? launch<FMT, false, false>(w, c, s) : launch<FMT, true, false>(w, c, s);
}

}  // namespace

hipError_t launch_few(const Weights &w, const Call &c, bool down, hipStream_t s) {
    switch (down ? w.down_type : w.up_type) {
    case Q8_0: return launch_type<Q8_0>(w, c, down, s);
    case Q4_0: return launch_type<Q4_0>(w, c, down, s);
    case Q4_K: return launch_type<Q4_K>(w, c, down, s);
    case Q6_K: return launch_type<Q6_K>(w, c, down, s);
    default: return hipErrorInvalidValue;
    }
}

}  // namespace ex
}  // namespace j4q
