// Products of tiles of up to 32 TM pairs with an expert's rows, weights as fp16 (experts.h).
//
// A workgroup of 4 waves has one tile of pairs; wave v has two groups of 32 rows of W, the same rows of gate and up or 64 rows of down,
// for all pairs: 2 TM v_mfma_f32_32x32x16_f16 accumulators. Each x' operand read from LDS feeds two MFMAs, and the activation needs no
// exchange. W is the first operand, so a lane holds 4 consecutive columns of the result for one pair. Two workgroups share a CU; or (TEAMS =
// 2) one of two such teams has it alone, which share W, with half of the tile's pairs each.
//
// K advances in stages of two 32-blocks. Lane (r, h) = (lane % 32, lane / 32) has block h of the stage: of row r of W, which it
// dequantizes, and of pair r's x'. MFMA p = 0..3 takes dword p of the codes and chunk p of the block layout. x' goes from
// global memory into one of two stage buffers (rows of 128 bytes, 16-byte chunk c of row r at slot c ^ ((r / 2) % 8)), W into units of
// two stages as in gemm_tile.h, whose WUnit and order of waits this is: X of stage i + 1 is issued behind the barrier of stage i,
// the unit after the next one at odd stages (Q8_0: units of one stage, at every one), and operands of MFMA p + 1 are dequantized under
// those of p.
//
// A weight is fp16(fma(code, s 2^pow, o 2^pow)), rounded once, with the row's power 2^pow that brings its largest magnitude into
// [2^13, 2^14) and leaves again in the epilogue: 11 bits down to 2^-27 of that. The code is an fp16 subnormal (a field masked out), so
// one v_fma_mix per weight does it. HL (fp32 x): hi + lo of both operands and three products, 22 bits;
// x's lo is stored 2^11 larger and meets W's hi 2^11 smaller (169 -> 174 us, 509 tokens of 32 Q4_0 experts).
//
// What bounds it are the matrix cores and the vector instructions that unpack W, whose times add, and the lines of W. 32744 pairs of 64
// experts 2048 x 1024, bf16: gate|up (Q4_K, tiles of 128) 287 us, 960 TFLOP/s, down (Q6_K, tiles of 96) 215 us, 640; 4086 pairs of 8 experts
// 4096 x 14336: 929 us, 1033 TFLOP/s, and 666 us, 721.
#include <type_traits>

#include "experts.h"
#include "gemm_tile.h"

namespace j4q {
namespace ex {
namespace {

using gw::dma16;
using gw::lds_barrier;
using gw::load_order;
using gw::wait_vm_lgkm0;
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef int32_t i32x4 __attribute__((ext_vector_type(4)));

// W of 4 waves of two groups of 32 rows in LDS, a unit at a time: two stages. Of Q4_K and Q6_K the codes; the scales of a superblock of
// four stages come with its first unit and lie apart, 16 bytes a row and Q6_K's d, once: a row's are read into registers before the
// next ones arrive. (What costs is the lines that a load touches, and each of these touches one a row.)
template <int FMT>
struct Unit : gt::WUnit<FMT, 8> {
    static constexpr int kStages = 2, kScales = 0;
};
template <int FMT>
struct SuperUnit : gt::WUnit<FMT, 8> {
    using Base = gt::WUnit<FMT, 8>;
    static constexpr int kStages = 2, kLoads = Base::kLoads - (FMT == Q6_K ? 2 : 1), kBytes = Base::kS, kSlot = FMT == Q6_K ? 768 : 1024, kScales = 8 * kSlot;
    uint32_t soff[FMT == Q6_K ? 2 : 1];
    __device__ __forceinline__ void init(const QMat &w, int nw, int wave_, int lane) {
        Base::init(w, nw, wave_, lane);
        // Q4_K: lane r < 32: row r's 16 bytes (the other lanes write zeros behind). Q6_K, for which LDS is short: dword L % 4 of 16 rows, twice.
#pragma unroll
        for (int j = 0; j < (FMT == Q6_K ? 2 : 1); j++) {
            const int n = nw + (FMT == Q6_K ? 16 * j + (lane >> 2) : lane);
            soff[j] = (FMT == Q6_K || lane < 32) && n < (int)w.rows ? (uint32_t)n * (uint32_t)(w.cols / 16) + (FMT == Q6_K ? 4u * (uint32_t)(lane & 3) : 0u) : kOob;
        }
    }
    __device__ __forceinline__ void load(int u, bool live, uint8_t *wb) const {
        const uint32_t uu = live ? (uint32_t)u : 0u;
#pragma unroll
        for (int j = 0; j < Base::QL; j++) dma16(this->qr, wb + (this->wave * Base::QL + j) * 1024, live ? this->qoff[j] : kOob, uu * (uint32_t)Base::QR);
        if constexpr (FMT == Q6_K) dma16(this->hr, wb + Base::kH + this->wave * 1024, live ? this->hoff : kOob, uu * 32u);
    }
    // The scales of unit u's superblock, u even.
    __device__ __forceinline__ void load_scales(int u, bool live, uint8_t *scales) const {
        uint8_t *const slot = scales + this->wave * kSlot;
        const uint32_t sb = live ? (uint32_t)u >> 1 : 0u;
        if constexpr (FMT == Q4_K) {
            dma16(this->sr, slot, live ? soff[0] : kOob, sb * 16u);
        } else {
            gw::dma4s(this->sr, slot, live ? soff[0] : kOob, sb * 16u);
            gw::dma4s(this->sr, slot + 256, live ? soff[1] : kOob, sb * 16u);
            gw::dma4(this->sr, slot + 512, live && this->doff != kOob ? (this->doff + sb * 2u) & ~3u : kOob);
        }
    }
};
template <>
struct Unit<Q4_K> : SuperUnit<Q4_K> {};
template <>
struct Unit<Q6_K> : SuperUnit<Q6_K> {};
// Q8_0: one stage, 64 bytes of codes a row (chunk c of row r at slot c ^ ((r / 4) % 4)) and a dword of scales; units of two stages
// would leave room for one workgroup a CU.
template <>
struct Unit<Q8_0> {
    static constexpr int kStages = 1, kScales = 0, QR = 64, QL = 2, kLoads = 3, kS = 8 * 32 * QR, kSlot = 256, kBytes = kS + 8 * kSlot;
    __amdgpu_buffer_rsrc_t qr, sr;
    uint32_t qoff[QL], soff;
    int wave;
    static __device__ __forceinline__ int swz(int row) { return (row >> 2) & 3; }
    __device__ __forceinline__ void init(const QMat &w, int nw, int wave_, int lane) {
        const int N = (int)w.rows, K = (int)w.cols;
        wave = wave_;
        qr = make_rsrc(w.qs, (uint64_t)N * (uint64_t)K);
        sr = make_rsrc(w.sc, (uint64_t)N * (uint64_t)(K / 16));
#pragma unroll
        for (int j = 0; j < QL; j++) {
            const int row = 16 * j + (lane >> 2), c = (lane & 3) ^ swz(row), n = nw + row;
            qoff[j] = n < N ? (uint32_t)n * (uint32_t)K + (uint32_t)c * 16u : kOob;
        }
        soff = lane < 32 && nw + lane < N ? (uint32_t)(nw + lane) * (uint32_t)(K / 16) : kOob;
    }
    __device__ __forceinline__ void load(int u, bool live, uint8_t *wb) const {
        const uint32_t uu = live ? (uint32_t)u : 0u;
#pragma unroll
        for (int j = 0; j < QL; j++) dma16(qr, wb + (wave * QL + j) * 1024, live ? qoff[j] : kOob, uu * 64u);
        gw::dma4s(sr, wb + kS + wave * kSlot, live ? soff : kOob, uu * 4u);
    }
};

// fp16(fma(c, s, o)) of two codes, and with HL what that leaves; `minus` is -1 in a register, with which the subtraction and its
// rounding are one v_fma_mix.
template <bool HL>
__device__ __forceinline__ void dequantize(uint32_t c, float s, float o, float minus, uint32_t &hi, uint32_t &lo) {
    const h2 v = __builtin_bit_cast(h2, c);
    const float a = __builtin_fmaf((float)v.x, s, o), b = __builtin_fmaf((float)v.y, s, o);
    const h2 h = {(_Float16)a, (_Float16)b};
    hi = __builtin_bit_cast(uint32_t, h);
    if constexpr (HL) {
        const h2 l = {(_Float16)__builtin_fmaf((float)h.x, minus, a), (_Float16)__builtin_fmaf((float)h.y, minus, b)};
        lo = __builtin_bit_cast(uint32_t, l);
    }
}

template <bool HL>
struct Operand {
    h8 hi, lo;
};
template <>
struct Operand<false> {
    h8 hi;
};

// One block of a row of W as it lies in LDS; scales s and offsets o of its elements 0..15 and 16..31.
template <int FMT>
struct Block {
    u32x4 q[FMT == Q8_0 ? 2 : 1];
    u32x2 hi;
    uint32_t s;
};
// The scales of a row's superblock.
struct Super {
    u32x4 s;
    uint32_t d;
};
struct Scale {
    float s[2], o[2];
};

// LDS of a workgroup with TM groups of 32 pairs.
template <int FMT, bool HL, int TM>
struct Lds {
    static constexpr int kPlane = 32 * TM * 128, kX = (HL ? 2 : 1) * kPlane;
};

// e with |v| < 2^e for the 64 values of a pair, whose halves lanes r and r + 32 have; values that are not finite do not count.
__device__ __forceinline__ int top_exponent(const f32x16 &a, const f32x16 &b) {
    auto both = [](float v) __attribute__((always_inline)) -> float {
        const uint32_t u = __builtin_bit_cast(uint32_t, v);
        const auto two = __builtin_amdgcn_permlane32_swap(u, u, false, false);
        return fmaxf(__builtin_bit_cast(float, (uint32_t)two[0]), __builtin_bit_cast(float, (uint32_t)two[1]));
    };
    float top = 0.f;
#pragma unroll
    for (int v = 0; v < 16; v++) top = fmaxf(fmaxf(top, fabsf(a[v])), fabsf(b[v]));
    top = both(top);
    if (__builtin_amdgcn_ballot_w64(!(top < __builtin_inff()))) {  // the wave as one
        top = 0.f;
#pragma unroll
        for (int v = 0; v < 16; v++) {
            top = fabsf(a[v]) < __builtin_inff() ? fmaxf(top, fabsf(a[v])) : top;
            top = fabsf(b[v]) < __builtin_inff() ? fmaxf(top, fabsf(b[v])) : top;
        }
        top = both(top);
    }
    return __builtin_amdgcn_frexp_expf(top);  // 0 of 0
}

// The products of one team of 4 waves; first and count: its pairs of the tile.
template <int FMT, bool HL, int TM, bool DOWN, int TEAMS>
__device__ __forceinline__ void run(const Weights &w, const Call &c, int expert, int first, int count, int chunk, int team, uint8_t *xs0, uint8_t *xs1, uint8_t *ws0,
                                    uint8_t *ws1, uint8_t *scales, uint8_t *team_place) {
    using U = Unit<FMT>;
    using L = Lds<FMT, HL, TM>;
    constexpr bool super = U::kScales != 0;
    constexpr int G = 2 / TEAMS, WL = G * U::kLoads, WS = WL + (FMT == Q4_K ? G : FMT == Q6_K ? 3 * G : 0),  // with scales; G: groups of W that a wave loads: its two, or one of the two it shares with the other team's
                   XL = (HL ? 2 : 1) * TM, QR = U::QR;
    const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6) & 3;
    const int r32 = lane & 31, h = lane >> 5;
    const int K = DOWN ? w.ffn : w.dim, N = DOWN ? w.dim : w.ffn, ns = K / 64, nsb = K / 256;
    // first row of W of each group
    const int n0 = DOWN ? 256 * chunk + 64 * wave : 128 * chunk + 32 * wave, n1 = DOWN ? n0 + 32 : n0;
    U unit[G];
    if constexpr (DOWN) {
        const QMat m = expert_of(w.down, FMT, expert, N);
#pragma unroll
        for (int g = 0; g < G; g++) {
            const int group = TEAMS == 2 ? team : g;
            unit[g].init(m, group ? n1 : n0, 2 * wave + group, lane);
        }
    } else {
#pragma unroll
        for (int g = 0; g < G; g++) {
            const int group = TEAMS == 2 ? team : g;
            unit[g].init(expert_of(group ? w.up : w.gate, FMT, expert, N), n0, 2 * wave + group, lane);
        }
    }
    const int32_t *const pow0 = (DOWN ? w.down_pow : w.gate_pow) + (int64_t)expert * N, *const pow1 = (DOWN ? w.down_pow : w.up_pow) + (int64_t)expert * N;
    float power[2];
    power[0] = n0 + r32 < N ? __builtin_ldexpf(1.f, pow0[n0 + r32]) : 1.f;
    power[1] = n1 + r32 < N ? __builtin_ldexpf(1.f, pow1[n1 + r32]) : 1.f;

    // X load j of this wave fills rows 8 (4 j + wave) .. + 7; lane L slot L % 8 of row 8 (4 j + wave) + L / 8.
    const _Float16 *const base = DOWN ? c.ha + (int64_t)first * K : c.xa;
    const uint64_t plane = DOWN ? (uint64_t)c.pairs * (uint64_t)K * 2u : (uint64_t)c.rows * (uint64_t)K * 2u;
    const uint64_t held = DOWN ? (uint64_t)count * (uint64_t)K * 2u : plane;
    const __amdgpu_buffer_rsrc_t xr = make_rsrc(base, held), xl = make_rsrc(HL ? (const uint8_t *)base + plane : (const uint8_t *)base, HL ? held : 0);
    uint32_t xoff[TM];
#pragma unroll
    for (int j = 0; j < TM; j++) {
        const int row = 8 * (4 * j + wave) + (lane >> 3), chunk16 = (lane & 7) ^ ((row >> 1) & 7);
        uint32_t at = kOob;
        if (row < count) at = (uint32_t)(DOWN ? row : row_of(c, c.order[first + row])) * (uint32_t)K * 2u + (uint32_t)chunk16 * 16u;
        xoff[j] = at;
    }
    auto load_x = [&](int i, uint8_t *xb) __attribute__((always_inline)) {
        const uint32_t so = i < ns ? (uint32_t)i * 128u : 0u;
#pragma unroll
        for (int j = 0; j < TM; j++) {
            dma16(xr, xb + (4 * j + wave) * 1024, i < ns ? xoff[j] : kOob, so);
            if constexpr (HL) dma16(xl, xb + L::kPlane + (4 * j + wave) * 1024, i < ns ? xoff[j] : kOob, so);
        }
    };
    auto load_w = [&](int u, uint8_t *wb) __attribute__((always_inline)) {
#pragma unroll
        for (int g = 0; g < G; g++) unit[g].load(u, U::kStages * u < ns, wb);
    };
    auto load_scales = [&](int u) __attribute__((always_inline)) {
        if constexpr (super) {
#pragma unroll
            for (int g = 0; g < G; g++) unit[g].load_scales(u, U::kStages * u < ns, scales);
        }
    };
    Super sup[2];
    auto read_super = [&](int group) __attribute__((always_inline)) {
        const uint8_t *const slot = scales + (2 * wave + group) * U::kSlot;
        sup[group].s = *reinterpret_cast<const u32x4 *>(slot + r32 * 16);
        if constexpr (FMT == Q6_K) sup[group].d = *reinterpret_cast<const uint32_t *>(slot + 512 + r32 * 4);
    };

    auto read_block = [&](int j, int group, const uint8_t *wb, Block<FMT> &o) __attribute__((always_inline)) {
        const int swz = U::swz(r32), blk = U::kStages == 2 ? 2 * (j & 1) + h : h, unit_row = 32 * (2 * wave + group) + r32;
        const uint8_t *const row = wb + unit_row * QR;
#pragma unroll
        for (int k = 0; k < (FMT == Q8_0 ? 2 : 1); k++) o.q[k] = *reinterpret_cast<const u32x4 *>(row + ((((FMT == Q8_0 ? 2 : 1) * blk + k) ^ swz) << 4));
        if constexpr (!super) o.s = *reinterpret_cast<const uint16_t *>(wb + U::kS + (2 * wave + group) * U::kSlot + r32 * (4 * U::kStages) + blk * 2);
        if constexpr (FMT == Q6_K) o.hi = *reinterpret_cast<const u32x2 *>(wb + U::kH + unit_row * 32 + blk * 8);
    };
    // Of block j, the Q-th stage of its superblock.
    auto decode_scale = [&](auto Q_, int j, int group, const Block<FMT> &b) __attribute__((always_inline)) -> Scale {
        constexpr float k24 = gt::kTwo24, k20 = gt::kTwo20;
        constexpr int Q = decltype(Q_)::value;
        const float pw = power[group];
        const Super &p = sup[group];
        Scale c;
        if constexpr (FMT == Q8_0) {
            const float d = half_bits_to_float(b.s) * pw;
            c.s[0] = c.s[1] = d * k24;
            c.o[0] = c.o[1] = -128.f * d;
        } else if constexpr (FMT == Q4_0) {
            const float d = half_bits_to_float(b.s) * pw;
            c.s[0] = d * k24;
            c.s[1] = d * k20;
            c.o[0] = c.o[1] = -8.f * d;
        } else if constexpr (FMT == Q4_K) {
            const int jsb = 2 * Q + h;
            const uint32_t sc = __builtin_amdgcn_ubfe(p.s[1], 4 * jsb, 4) | (__builtin_amdgcn_ubfe(p.s[3], 2 * jsb, 2) << 4);
            const uint32_t mn = __builtin_amdgcn_ubfe(p.s[2], 4 * jsb, 4) | (__builtin_amdgcn_ubfe(p.s[3], 16 + 2 * jsb, 2) << 4);
            const float d = half_bits_to_float(p.s[0] & 0xFFFFu) * pw * (float)sc;
            c.s[0] = d * k24;
            c.s[1] = d * k20;
            c.o[0] = c.o[1] = -(half_bits_to_float(p.s[0] >> 16) * pw * (float)mn);
        } else {
            const int n = (group ? n1 : n0) + r32;
            const uint32_t odd = ((uint32_t)n * (uint32_t)nsb + (uint32_t)(j >> 2)) & 1u;  // an expert's rows are a multiple of 64
            const float d = half_bits_to_float(odd ? p.d >> 16 : p.d & 0xFFFFu) * pw;
            const uint32_t two = h ? p.s[Q] >> 16 : p.s[Q];
            const float da = d * (float)(int8_t)(two & 0xFFu), db = d * (float)(int8_t)(two >> 8 & 0xFFu);
            c.s[0] = da * k24;
            c.o[0] = -32.f * da;
            c.s[1] = db * k20;
            c.o[1] = -32.f * db;
        }
        return c;
    };
    float minus = -1.f;
    asm("" : "+v"(minus));
    // Operand p of a block.
    auto operand = [&](const Block<FMT> &b, const Scale &c, int p, Operand<HL> &out) __attribute__((always_inline)) {
        uint32_t part[4];
        if constexpr (FMT == Q8_0) {
            const uint32_t u = b.q[0][p] ^ 0x80808080u, v = b.q[1][p] ^ 0x80808080u;
            part[0] = u & 0x00FF00FFu;
            part[1] = u >> 8 & 0x00FF00FFu;
            part[2] = v & 0x00FF00FFu;
            part[3] = v >> 8 & 0x00FF00FFu;
        } else {
            const uint32_t v = b.q[0][p], t = v >> 8;
            part[0] = v & 0x000F000Fu;
            part[1] = t & 0x000F000Fu;
            part[2] = v & 0x00F000F0u;
            part[3] = t & 0x00F000F0u;
            if constexpr (FMT == Q6_K) {
                const uint32_t raw = b.hi[p >> 1], hw = p & 1 ? __builtin_amdgcn_alignbit(raw, raw, 8) : raw, u = hw >> 2;
                part[0] |= hw & 0x00300030u;
                part[1] |= u & 0x00300030u;
                part[2] |= hw & 0x03000300u;
                part[3] |= u & 0x03000300u;
            }
        }
        u32x4 hi, lo;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            uint32_t x = 0, y = 0;
            dequantize<HL>(part[k], c.s[k >> 1], c.o[k >> 1], minus, x, y);
            hi[k] = x;
            lo[k] = y;
        }
        out.hi = __builtin_bit_cast(h8, hi);
        if constexpr (HL) out.lo = __builtin_bit_cast(h8, lo);
    };

    f32x16 acc[2][TM];
#pragma unroll
    for (int t = 0; t < TM; t++) acc[0][t] = acc[1][t] = f32x16{};
    const int xrow = r32 * 128, xsw = (r32 >> 1) & 7;
    auto read_x = [&](const uint8_t *xb, int p, Operand<HL> (&a)[TM]) __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < TM; t++) {
            const uint8_t *const at = xb + t * 32 * 128 + xrow + (((4 * h + p) ^ xsw) << 4);
            a[t].hi = *reinterpret_cast<const h8 *>(at);
            if constexpr (HL) a[t].lo = *reinterpret_cast<const h8 *>(at + L::kPlane);
        }
    };
    // vector instructions behind an MFMA; two teams' down spills with 8 (8192 pairs of Q6_K gate and up, fp32: 866 us with 7, 843 with 8)
    constexpr int kShadow = HL ? (TEAMS == 2 && !DOWN ? 8 : 7) : TM >= 4 ? 5 : TM == 3 ? 7 : TM == 2 ? 9 : 18;
    Block<FMT> blk[2][2];  // [stage parity][group]
    Scale sc[2][2];
    Operand<HL> b[2][2];   // of MFMA p and p + 1
    auto stage = [&](auto S_, int i) __attribute__((always_inline)) {
        constexpr int S = decltype(S_)::value, cur = S & 1;
        uint8_t *const xb = cur ? xs1 : xs0, *const xn = cur ? xs0 : xs1;
        using Next = std::integral_constant<int, (S + 1) % 4>;
        constexpr bool pairs = U::kStages == 2;
        constexpr int ur = pairs ? (S + 1) / 2 % 2 : (S + 1) % 2, un = pairs ? (S + 3) / 2 % 2 : S % 2;
        uint8_t *const wc = ur ? ws1 : ws0, *const wn = un ? ws1 : ws0;
        wait_vm_lgkm0<!pairs || S % 2 ? 0 : S == 0 ? WL : WS>();  // the newest unit of W, at stage 2 with its scales, is under way
        lds_barrier();
        Operand<HL> a[2][TM];
        read_x(xb, 0, a[0]);
        read_block(i + 1, 0, wc, blk[cur ^ 1][0]);
        read_block(i + 1, 1, wc, blk[cur ^ 1][1]);
        if constexpr (super && S == 3) {
            read_super(0);
            read_super(1);
        }
        load_x(i + 1, xn);
        load_order();  // X first: the wait at an even stage leaves the newest unit of W outstanding
        if constexpr (!pairs) load_w(i + 2, wn);
        else if constexpr (S % 2 == 1) load_w((i + 3) / 2, wn);
        if constexpr (S == 1) load_scales((i + 3) / 2);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int p = 0; p < 4; p++) {
            if (p < 3) read_x(xb, p + 1, a[(p + 1) & 1]);
            if (p == 1) {
                sc[cur ^ 1][0] = decode_scale(Next{}, i + 1, 0, blk[cur ^ 1][0]);
                sc[cur ^ 1][1] = decode_scale(Next{}, i + 1, 1, blk[cur ^ 1][1]);
            }
#pragma unroll
            for (int g = 0; g < 2; g++) {
                h8 over;  // x's lo is stored kLow larger: 11 bits of W down to 2^-16 of the row's largest
                if constexpr (HL) over = b[p & 1][g].hi * (_Float16)(1.f / kLow);
#pragma unroll
                for (int t = 0; t < TM; t++) {
                    if constexpr (HL) {
                        acc[g][t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(b[p & 1][g].lo, a[p & 1][t].hi, acc[g][t], 0, 0, 0);
                        acc[g][t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(over, a[p & 1][t].lo, acc[g][t], 0, 0, 0);
                    }
                    acc[g][t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(b[p & 1][g].hi, a[p & 1][t].hi, acc[g][t], 0, 0, 0);
                }
                if (p < 3) operand(blk[cur][g], sc[cur][g], p + 1, b[(p + 1) & 1][g]);
                else operand(blk[cur ^ 1][g], sc[cur ^ 1][g], 0, b[0][g]);
            }
        }
        // vector instructions in the shadow of every MFMA, rather than behind a run of them
#pragma unroll
        for (int k = 0; k < 8 * TM * (HL ? 3 : 1); k++) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x002, kShadow, 0);
        }
        // computed here, between the MFMAs, although the last stage does not use it
        asm volatile("" : "+v"(b[0][0].hi), "+v"(b[0][1].hi));
    };

    load_w(0, ws0);
    load_scales(0);
    load_order();
    load_x(0, xs0);
    load_order();
    load_w(1, ws1);
    wait_vm_lgkm0<XL + WL>();
    if constexpr (TEAMS == 2) lds_barrier();  // half of its W came by the other team
    else asm volatile("" ::: "memory");
#pragma unroll
    for (int g = 0; g < 2; g++) {
        read_block(0, g, ws0, blk[0][g]);
        if constexpr (super) read_super(g);
        sc[0][g] = decode_scale(std::integral_constant<int, 0>{}, 0, g, blk[0][g]);
        operand(blk[0][g], sc[0][g], 0, b[0][g]);
    }
#define J4Q_STAGE(S) stage(std::integral_constant<int, S>{}, i + S);
    int i = 0;
    for (; i + 4 <= ns; i += 4) {
        J4Q_STAGE(0) J4Q_STAGE(1) J4Q_STAGE(2) J4Q_STAGE(3)
    }
    if constexpr (FMT == Q8_0 || FMT == Q4_0) {
        if (i < ns) {
            J4Q_STAGE(0)
            if (i + 1 < ns) {
                J4Q_STAGE(1)
                if (i + 2 < ns) J4Q_STAGE(2)
            }
        }
    }
#undef J4Q_STAGE
    __builtin_amdgcn_s_waitcnt(0);  // no LDS load outlives the workgroup

    if (TEAMS == 2 && count == 0) {
        if constexpr (DOWN) __syncthreads();
        return;
    }
    // Element v of acc[g][t]: row n + 8 (v / 4) + 4 h + v % 4 of the group, pair 32 t + r32.
    i32x4 p0[4], p1[4];
#pragma unroll
    for (int q = 0; q < 4; q++) {
        const int a = n0 + 8 * q + 4 * h, e = n1 + 8 * q + 4 * h;
        p0[q] = a < N ? *reinterpret_cast<const i32x4 *>(pow0 + a) : i32x4{};
        p1[q] = e < N ? *reinterpret_cast<const i32x4 *>(pow1 + e) : i32x4{};
    }
    if constexpr (DOWN) {
        // Through LDS, 32 pairs at a time, so that whole lines are stored: a pair's 64 columns of this wave are 8 chunks of 16 bytes of
        // fp16, or 16 of fp32; chunk k of pair p at k ^ (p % 8).
        __syncthreads();  // all waves have read their W and x'
        // 8 KiB a wave: in the buffers of W, of two teams in those of x'
        uint8_t *const place = TEAMS == 2 ? team_place : (wave < 2 ? ws0 : ws1) + (wave & 1) * 8192;
        constexpr int C = HL ? 16 : 8;  // chunks of a pair
#pragma unroll
        for (int t = 0; t < TM; t++) {
            const int m = 32 * t + r32;
            const int pair = c.order[first + (m < count ? m : 0)], token = row_of(c, pair), hp = h_pow(w, expert, c.x_norm[token]);
            const float weight = HL ? c.weights[pair] : 1.f;
            int up = -hp;
            if constexpr (!HL) {
#pragma unroll
                for (int v = 0; v < 16; v++) {
                    acc[0][t][v] = __builtin_ldexpf(acc[0][t][v], -p0[v >> 2][v & 3]);
                    acc[1][t][v] = __builtin_ldexpf(acc[1][t][v], -p1[v >> 2][v & 3]);
                }
                up = 14 - top_exponent(acc[0][t], acc[1][t]);
                if (h == 0 && m < count && n0 < N) c.part_pow[(int64_t)pair * (N / 64) + n0 / 64] = -hp - up;
            }
#pragma unroll
            for (int g = 0; g < 2; g++)
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    f32x4 v;
#pragma unroll
                    for (int j = 0; j < 4; j++) v[j] = HL ? __builtin_ldexpf(acc[g][t][4 * q + j] * weight, up - (g ? p1[q][j] : p0[q][j])) : __builtin_ldexpf(acc[g][t][4 * q + j], up);
                    if constexpr (HL) *reinterpret_cast<f32x4 *>(place + r32 * 256 + (((8 * g + 2 * q + h) ^ (r32 & 7)) << 4)) = v;
                    else *reinterpret_cast<h4 *>(place + r32 * 128 + (((4 * g + q) ^ (r32 & 7)) << 4) + 8 * h) = __builtin_convertvector(v, h4);
                }
            asm volatile("" ::: "memory");  // a wave's own place, whose operations are in order
#pragma unroll
            for (int i = 0; i < C / 2; i++) {
                const int p = (64 / C) * i + lane / C, k = lane % C, n = n0 + (HL ? 4 : 8) * k;
                const u32x4 v = *reinterpret_cast<const u32x4 *>(place + p * (16 * C) + ((k ^ (p & 7)) << 4));
                if (32 * t + p >= count || n >= N) continue;
                const int64_t at = (int64_t)c.order[first + 32 * t + p] * N + n;
                if constexpr (HL) *reinterpret_cast<u32x4 *>(c.part + at) = v;
                else *reinterpret_cast<u32x4 *>((_Float16 *)c.part + at) = v;
            }
            asm volatile("" ::: "memory");
        }
        return;
    }
#pragma unroll
    for (int t = 0; t < TM; t++) {
        const int m = 32 * t + r32;
        if (m >= count || n0 >= N) continue;
        const int pair = c.order[first + m], token = row_of(c, pair), hp = h_pow(w, expert, c.x_norm[token]), e = -c.x_pow[token];
        _Float16 *const out = c.ha + (int64_t)(first + m) * N + n0;
        const int64_t lo = (int64_t)c.pairs * N;
#pragma unroll
        for (int k = 0; k < 2; k++) {  // chunk 2 k + h of the block: elements of q = k, then of q = 2 + k
            h8 hi, rest;
#pragma unroll
            for (int s = 0; s < 8; s++) {
                const int q = k + 2 * (s >> 2), j = (s & 1) << 1 | (s >> 1 & 1);
                const float gv = __builtin_ldexpf(acc[0][t][4 * q + j], e - p0[q][j]), uv = __builtin_ldexpf(acc[1][t][4 * q + j], e - p1[q][j]);
                const float v = __builtin_ldexpf(activate(gv, w.act) * uv, hp);
                hi[s] = (_Float16)v;
                rest[s] = (_Float16)((v - (float)hi[s]) * kLow);
            }
            *reinterpret_cast<h8 *>(out + 8 * (2 * k + h)) = hi;
            if constexpr (HL) *reinterpret_cast<h8 *>(out + lo + 8 * (2 * k + h)) = rest;
        }
    }
}

// grid: tiles * chunks, rounded up to whole eighths; a chunk is 128 columns of the result (down: 256).
template <int FMT, bool HL, int TM, bool DOWN, int TEAMS>
__global__ void __launch_bounds__(256 * TEAMS, 2)
experts_many(Weights w, Call c) {
    constexpr int kX = Lds<FMT, HL, TM>::kX, kW = Unit<FMT>::kBytes, kS = Unit<FMT>::kScales;
    static_assert((2 * (TEAMS * kX + kW) + kS) * (2 / TEAMS) <= 163840, "a CU's LDS");
    static_assert(TEAMS == 2 ? kX >= 16384 : kW >= 16384, "room for the waves' results");
    // arrays of their own: what tells the compiler that a read of one need not wait for loads into another
    __shared__ __attribute__((aligned(1024))) uint8_t xs0[TEAMS * kX], xs1[TEAMS * kX];
    __shared__ __attribute__((aligned(1024))) uint8_t ws0[kW], ws1[kW];
    __shared__ __attribute__((aligned(1024))) uint8_t scales[kS ? kS : 16];
    const int N = DOWN ? w.dim : w.ffn, chunks = DOWN ? (N + 255) / 256 : (N + 127) / 128, tiles = (DOWN ? c.down : c.up).count[0];
    // Workgroup b runs on XCD b % 8, and each XCD takes a contiguous range, down groups of 4 tiles of pairs: most often of one
    // expert, whose rows of W they share in the XCD's L2.
    const int total = tiles * chunks, per = (total + 7) / 8, at = (int)(blockIdx.x % 8) * per + (int)(blockIdx.x / 8);
    if ((int)(blockIdx.x / 8) >= per || at >= total) return;
    const int mg = at / (4 * chunks), gm = tiles - 4 * mg < 4 ? tiles - 4 * mg : 4, rem = at - 4 * mg * chunks, chunk = rem / gm;
    const Tile tile = (DOWN ? c.down : c.up).tile[4 * mg + rem % gm];
    const int expert = __builtin_amdgcn_readfirstlane(tile.expert), all = __builtin_amdgcn_readfirstlane(tile.count);
    // the groups of 32 pairs, fewer in an expert's last tile, half of them for each team
    const int team = TEAMS == 2 ? __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 8) : 0, groups = ((all + 31) / 32 + TEAMS - 1) / TEAMS;
    const int skip = 32 * groups * team, first = __builtin_amdgcn_readfirstlane(tile.first) + skip;
    const int left = all - skip < 0 ? 0 : all - skip, count = left < 32 * groups ? left : 32 * groups;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    uint8_t *const place = (wave < 4 ? xs0 : xs1) + (wave & 3) * 8192;
#define J4Q_RUN(T) run<FMT, HL, (TM < T ? TM : T), DOWN, TEAMS>(w, c, expert, first, count, chunk, team, xs0 + team * kX, xs1 + team * kX, ws0, ws1, scales, place)
    if (groups >= TM) J4Q_RUN(TM);
    else if (TM > 3 && groups == 3) J4Q_RUN(3);
    else if (TM > 2 && groups == 2) J4Q_RUN(2);
    else J4Q_RUN(1);
#undef J4Q_RUN
}

template <int FMT, bool DOWN>
hipError_t launch_type(const Weights &w, const Call &c, hipStream_t s) {
    const int N = DOWN ? w.dim : w.ffn, chunks = DOWN ? (N + 255) / 256 : (N + 127) / 128;
    const Tiles &tiles = DOWN ? c.down : c.up;
    const int64_t total = ((int64_t)tiles.most * chunks + 7) / 8 * 8;
    if (total > 0xffffff) return hipErrorInvalidValue;
    const dim3 grid((unsigned)total);
    bool launched = false;
#define J4Q_MANY(HL, TM, TEAMS)                                                    \
    if (c.half == !HL && tiles.rows == 32 * TM * TEAMS) {                          \
        experts_many<FMT, HL, TM, DOWN, TEAMS><<<grid, 256 * TEAMS, 0, s>>>(w, c); \
        launched = true;                                                           \
    }
    J4Q_MANY(false, 1, 1)
    J4Q_MANY(false, 2, 1)
    if constexpr (FMT == Q6_K) {
        J4Q_MANY(false, 3, 1)
    } else {
        J4Q_MANY(false, 4, 1)
    }
    J4Q_MANY(true, 1, 1)
    if constexpr (FMT == Q6_K) {
        J4Q_MANY(true, 2, 2)
    } else {
        J4Q_MANY(true, 2, 1)
    }
#undef J4Q_MANY
    if (!launched) return hipErrorInvalidValue;
    return hipGetLastError();
}

}  // namespace

// `each`: pairs per expert on average. The most pairs a tile with which two workgroups' LDS fit a CU: they run out of phase, one's
// MFMAs under the other's barriers (two teams in one workgroup of bf16, tiles of 256: 1737 -> 1916 us). With Q6_K and fp32 those are tiles
// of 32, and two teams with 64 each are faster from some 200 pairs an expert on (8192 pairs of 32 experts, 2048 x 2048: 976 -> 850 us; 1024
// of 8: 184 -> 195). bf16 x, 4 of 32 experts 2048 x 1024 of Q4_K, 50 pairs each: tiles of 32 104 us, of 64 93; 80 each: of 64 89, of
// 128 107; 110 each: 123, 111.
int rows_many(int type, bool half, int each) {
    if (!half && type == Q6_K) return each < 192 ? 32 : 128;
    if (each < 40) return 32;
    if (each < 96 || !half) return 64;
    return type == Q6_K ? 96 : 128;
}

hipError_t launch_many(const Weights &w, const Call &c, bool down, hipStream_t s) {
    switch (down ? w.down_type : w.up_type) {
    case Q8_0: return down ? launch_type<Q8_0, true>(w, c, s) : launch_type<Q8_0, false>(w, c, s);
    case Q4_0: return down ? launch_type<Q4_0, true>(w, c, s) : launch_type<Q4_0, false>(w, c, s);
    case Q4_K: return down ? launch_type<Q4_K, true>(w, c, s) : launch_type<Q4_K, false>(w, c, s);
    case Q6_K: return down ? launch_type<Q6_K, true>(w, c, s) : launch_type<Q6_K, false>(w, c, s);
    default: return hipErrorInvalidValue;
    }
}

}  // namespace ex
}  // namespace j4q
