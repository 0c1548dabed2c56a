// Products of tiles of up to 16 pairs (fp32: 8) with an expert's rows, exact codes (experts_codes.h).
//
// Bound by the stream of W. What stood in its way was not the memory but the CU's path to it, which takes a cache line every four
// clocks whatever is used of it: with operands loaded straight into registers (64 bytes of 16 rows a load, scales dword by dword, x'
// by every wave for itself) gate|up of 48 tokens x 6 of 64 Q8_0 experts 2048 x 1408 stood at 3.0 TB/s. Here all of it comes as whole
// lines into LDS (buffer_load ... lds, no registers held while it is on its way), x' once for a workgroup.
//
// A workgroup of 8 waves has one tile of pairs; wave v has 16 rows of W over all of K: of gate (v < 4) or up, of the same 64 columns
// of the result, or of down's 128. K advances in stages of 256 columns (Q8_0: 128) through a ring of D buffers: at stage i a wave
// waits for its own loads of stage i, meets the others, issues stage i + D - 1 into the buffer of stage i - 1, and multiplies.
// Two workgroups share a CU. 16-byte chunks lie swizzled: chunk c of row r of W at c ^ ((r / 2) % 4), of x' at c ^ r, so that the rows
// of an operand read fall on distinct banks (of W, two on each: with three bits of the row the places of 8 blocks in 3 buffers would not
// fit the registers).
//
// The stream of W bounds it: 48 tokens, 6 of 64 experts 2048 x 1408 of Q8_0, bf16: gate|up 68 us, 5.7 TB/s, down 39 us, 5.0 TB/s.
#include <type_traits>

#include "experts_codes.h"
#include "gemm_wide.h"

namespace j4q {
namespace ex {
namespace {

using gmf::lane_off;  // (a select, no branch)
using gw::dma16;
using gw::dma4s;
using gw::lds_barrier;
using gw::wait_vm_lgkm0;

constexpr int kWaves = 8;

template <int FMT>
struct Ring {
    static constexpr int kDepth = FMT == Q6_K ? 2 : 3;
    static constexpr int kCols = FMT == Q8_0 ? 128 : 256, kBlocks = kCols / 32;  // of a stage
    // a wave's part of a buffer: codes, Q6_K's high bits, scale words, Q6_K's d
    static constexpr int kHigh = 2048, kScale = kHigh + (FMT == Q6_K ? 1024 : 0), kD = kScale + 256, kWave = kD + (FMT == Q6_K ? 256 : 0);
    static constexpr int kX = kWaves * kWave, kBytes = kX + 8192;  // x' (Q8_0: half of it; the other waves' loads of nothing fill the rest)
    static constexpr int kLoads = 4 + (FMT == Q6_K ? 2 : 0);       // of a wave and stage
};

// A wave's 16 rows of W.
template <int FMT>
struct Stream {
    using R = Ring<FMT>;
    __amdgpu_buffer_rsrc_t qr, hr, sr, dr;
    uint32_t qoff[2], hoff, soff, doff;
    int K;
    __device__ __forceinline__ void init(const QMat &m, int row0, int lane, bool ok) {
        K = (int)m.cols;
        const uint64_t rows = (uint64_t)m.rows, k = (uint64_t)K;
        const uint32_t qrow = FMT == Q8_0 ? (uint32_t)K : (uint32_t)(K / 2);
        qr = make_rsrc(m.qs, rows * qrow);
        sr = make_rsrc(m.sc, rows * (k / 16));
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const int r = 8 * j + (lane >> 3), c = (lane & 7) ^ ((r >> 1) & 3);
            qoff[j] = ok ? (uint32_t)(row0 + r) * qrow + (uint32_t)c * 16u : kOob;
        }
        const uint32_t r = (uint32_t)(row0 + (lane >> 2)), part = (uint32_t)lane & 3u;
        soff = ok && (FMT != Q8_0 || part < 2) ? r * (uint32_t)(K / 16) + 4u * part : kOob;
        if constexpr (FMT == Q6_K) {
            hr = make_rsrc(m.qh, rows * (k / 4));
            dr = make_rsrc(m.d, rows * (k / 128));
            hoff = ok ? r * (uint32_t)(K / 4) + ((part ^ (r >> 1 & 1u)) * 16u) : kOob;
            doff = ok && lane < 16 ? (uint32_t)(row0 + lane) * (uint32_t)(K / 128) : kOob;
        }
    }
    // In two parts, each with the other half of the stage before it.
    __device__ __forceinline__ void load(int part, int i, bool live, uint8_t *at, int lane) const {
        const uint32_t u = live ? (uint32_t)i : 0u;
        dma16(qr, at + 1024 * part, lane_off(qoff[part], live), u * 128u);
        if (part == 0) return;
        if constexpr (FMT == Q6_K) dma16(hr, at + R::kHigh, lane_off(hoff, live), u * 64u);
        // a dword of two blocks' scales (Q8_0, Q4_0) behind the row's last block: nothing
        const bool in = (FMT == Q4_K) | (FMT == Q6_K) | ((int)(u * R::kBlocks) + 2 * (lane & 3) < K / 32);
        dma4s(sr, at + R::kScale, lane_off(soff, live & in), u * (R::kBlocks * 2u));
        if constexpr (FMT == Q6_K) dma4s(dr, at + R::kD, lane_off((doff + 2u * u) & ~3u, live & (doff != kOob)), 0u);
    }
};

// grid: (ceil(N / 64) or down ceil(N / 128) * splits, tiles over y and z).
template <int FMT, bool HL, bool DOWN>
__global__ void __launch_bounds__(kWaves * 64, 4)
experts_few(Weights w, Call c) {
    using R = Ring<FMT>;
    constexpr int D = R::kDepth;
    static_assert(2 * D * R::kBytes <= 163840, "two workgroups' LDS");
    __shared__ __attribute__((aligned(1024))) uint8_t b0[R::kBytes], b1[R::kBytes], b2[D == 3 ? R::kBytes : 16];
    const int at = (int)(blockIdx.z * gridDim.y + blockIdx.y);
    const Tiles &tiles = DOWN ? c.down : c.up;
    if (at >= tiles.most) return;
    const Tile tile = tiles.tile[at];  // (with the count, not behind it)
    if (at >= tiles.count[0]) return;
    const int expert = __builtin_amdgcn_readfirstlane(tile.expert), count = __builtin_amdgcn_readfirstlane(tile.count),
              first = __builtin_amdgcn_readfirstlane(tile.first);
    const int lane = (int)threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int n = lane & 15, g = lane >> 4;
    const int K = DOWN ? w.ffn : w.dim, N = DOWN ? w.dim : w.ffn, all = (K + R::kCols - 1) / R::kCols;
    // down: K in c.splits ranges of whole stages
    const int chunks = DOWN ? (N + 127) / 128 : (int)gridDim.x, split = DOWN ? (int)blockIdx.x / chunks : 0, chunk = (int)blockIdx.x - split * chunks;
    const int each = DOWN ? (all + c.splits - 1) / c.splits : all, from = split * each, ns = all < from + each ? all : from + each;
    const int row0 = DOWN ? 128 * chunk + 16 * wave : 64 * chunk + 16 * (wave & 3);
    Stream<FMT> s;
    s.init(expert_of(DOWN ? w.down : wave < 4 ? w.gate : w.up, FMT, expert, N), row0, lane, row0 < N);

    // x' of a stage: row r = 2 wave + lane / 32 (Q8_0: 4 wave + lane / 16) of the operand: pair r, with HL pair r % 8 and its hi or lo part
    constexpr int XC = R::kCols / 8;  // chunks of a row
    uint32_t xoff = kOob, xchunk = 0;
    const int64_t plane = (int64_t)(DOWN ? c.pairs : c.rows) * K;
    const __amdgpu_buffer_rsrc_t xr = make_rsrc(DOWN ? c.ha + (int64_t)first * K : c.xa, (uint64_t)((HL ? 2 : 1) * plane - (DOWN ? (int64_t)first * K : 0)) * 2u);
    {
        const int r = (64 / XC) * wave + lane / XC, m = HL ? r & 7 : r;
        xchunk = (uint32_t)((lane % XC) ^ (r & 15));
        if (r < 16 && m < count) {
            const int64_t at_row = (int64_t)(DOWN ? m : row_of(c, c.order[first + m])) * K + (HL && r >= 8 ? plane : 0);
            xoff = (uint32_t)at_row * 2u + xchunk * 16u;
        }
    }
    auto load = [&](int part, int i, uint8_t *buf) __attribute__((always_inline)) {
        const bool live = i < ns;
        const uint32_t u = live ? (uint32_t)i : 0u;
        s.load(part, i, live, buf + wave * R::kWave, lane);
        if (part == 0) dma16(xr, buf + R::kX + 1024 * wave, lane_off(xoff, live & ((int)(u * (R::kCols / 8) + xchunk) < K / 8)), u * (R::kCols * 2u));
    };

    f32x4 acc = {}, low = {};
    const uint32_t one = or_one();
    // Places in a buffer of what this lane reads of four blocks; the next four lie 64 (W) and 256 bytes (x') behind.
    uint32_t xat[4], wat[4];
#pragma unroll
    for (int k = 0; k < 4; k++) {
        xat[k] = (uint32_t)(R::kX + n * (R::kCols * 2) + (((4 * k + g) ^ n) << 4));
        wat[k] = (uint32_t)(wave * R::kWave + n * 128 + ((k ^ (n >> 1 & 3)) << 4) + 4 * g);
    }
    uint32_t hat[2];
#pragma unroll
    for (int k = 0; k < 2; k++) hat[k] = (uint32_t)(wave * R::kWave + R::kHigh + n * 64 + ((k ^ (n >> 1 & 1)) << 4) + 4 * (g >> 1));
    const uint32_t sat = (uint32_t)(wave * R::kWave + R::kScale + n * 16);
    auto stage = [&](int i, const uint8_t *buf, uint8_t *next) __attribute__((always_inline)) {
        wait_vm_lgkm0<(D - 2) * R::kLoads>();
        lds_barrier();
        Raw<FMT> r;
        r.s = *reinterpret_cast<const u32x4 *>(buf + sat);
        if constexpr (FMT == Q6_K) {
            const uint32_t d = *reinterpret_cast<const uint32_t *>(buf + wave * R::kWave + R::kD + n * 4);
            r.d = ((row0 + n) * (K / 256) + i) & 1 ? d >> 16 : d & 0xFFFFu;
        }
        auto part = [&](auto half_) __attribute__((always_inline)) {
            constexpr int half = decltype(half_)::value, B = R::kBlocks / 2;
            Operands<FMT> a;
#pragma unroll
            for (int k = 0; k < B; k++) a.x[k] = *reinterpret_cast<const h8 *>(buf + xat[(B * half + k) & 3] + 256 * ((B * half + k) >> 2));
#pragma unroll
            for (int k = 0; k < 4; k++) r.v[k] = *reinterpret_cast<const uint32_t *>(buf + wat[k] + 64 * half);
            if constexpr (FMT == Q6_K) {
#pragma unroll
                for (int k = 0; k < 4; k += 2) {
                    const uint8_t *const at = buf + hat[k / 2] + 32 * half;
                    const uint32_t u = *reinterpret_cast<const uint32_t *>(at), v = *reinterpret_cast<const uint32_t *>(at + 8);
                    r.h[k] = __builtin_amdgcn_alignbit(u, u, (uint32_t)(g & 1) * 8u);
                    r.h[k + 1] = __builtin_amdgcn_alignbit(v, v, (uint32_t)(g & 1) * 8u);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
            load(half, i + D - 1, next);
            __builtin_amdgcn_sched_barrier(0);
            multiply<FMT>(r, a, half, g, one, acc, low);
            __builtin_amdgcn_sched_barrier(0);
        };
        part(std::integral_constant<int, 0>{});
        part(std::integral_constant<int, 1>{});
    };
#pragma unroll
    for (int k = 0; k < 2 * (D - 1); k++) {
        load(k & 1, from + (k >> 1), k < 2 ? b0 : b1);
        __builtin_amdgcn_sched_barrier(0);
    }
    for (int i = from; i < ns; i += D) {
        if constexpr (D == 3) {
            stage(i, b0, b2);
            stage(i + 1, b1, b0);  // behind the last stage: zeros
            stage(i + 2, b2, b1);
        } else {
            stage(i, b0, b1);
            stage(i + 1, b1, b0);
        }
    }
    __builtin_amdgcn_s_waitcnt(0);  // no load into LDS outlives its buffer
    __syncthreads();
    float *const red = reinterpret_cast<float *>(b0);
    static_assert(R::kBytes >= kWaves * 1024, "results in a buffer");
#pragma unroll
    for (int j = 0; j < 4; j++) red[wave * 256 + (4 * g + j) * 16 + n] = acc[j] - low[j];
    __syncthreads();
    auto value = [&](int tile16, int o) __attribute__((always_inline)) -> float {
        const float *const v = red + tile16 * 256 + o;
        return HL ? __builtin_fmaf(v[128], 1.f / kLow, v[0]) : v[0];
    };
    constexpr int kOut = HL ? 128 : 256, COLS = DOWN ? kWaves : kWaves / 2;
    for (int o = (int)threadIdx.x; o < COLS * kOut; o += kWaves * 64) {
        const int ct = o / kOut, i = o % kOut, q = i >> 4, col = 16 * (COLS * chunk + ct) + (i & 15);
        if (q >= count || col >= N) continue;
        const int pair = c.order[first + q], token = row_of(c, pair), pow = h_pow(w, expert, c.x_norm[token]);
        if constexpr (DOWN) {
            c.part[((int64_t)split * c.pairs + pair) * N + col] = __builtin_ldexpf(value(ct, i) * c.weights[pair], -pow);  // the weight first: the product alone may not fit
        } else {
            const int e = -c.x_pow[token];
            const float h = __builtin_ldexpf(activate(__builtin_ldexpf(value(ct, i), e), w.act) * __builtin_ldexpf(value(4 + ct, i), e), pow);
            const _Float16 hi = (_Float16)h;
            _Float16 *const out = c.ha + (int64_t)(first + q) * w.ffn + slot_of(col);
            *out = hi;
            if constexpr (HL) out[(int64_t)c.pairs * w.ffn] = (_Float16)((h - (float)hi) * kLow);
        }
    }
}

template <int FMT, bool HL, bool DOWN>
hipError_t launch(const Weights &w, const Call &c, hipStream_t s) {
    const int N = DOWN ? w.dim : w.ffn, cols = DOWN ? 128 : 64;
    const int tiles = (DOWN ? c.down : c.up).most, y = tiles < 32768 ? tiles : 32768;
    const dim3 grid((unsigned)((N + cols - 1) / cols * (DOWN ? c.splits : 1)), (unsigned)y, (unsigned)((tiles + y - 1) / y));
    experts_few<FMT, HL, DOWN><<<grid, kWaves * 64, 0, s>>>(w, c);
    return hipGetLastError();
}

template <int FMT>
hipError_t launch_type(const Weights &w, const Call &c, bool down, hipStream_t s) {
    if (down) return c.half ? launch<FMT, false, true>(w, c, s) : launch<FMT, true, true>(w, c, s);
    return c.half ? launch<FMT, false, false>(w, c, s) : launch<FMT, true, false>(w, c, s);
}

}  // namespace

// Three workgroups for each CU of an MI355X (a constant, so that results do not depend on the device), of at least 1024 columns (5
// tokens through 2 of 8 experts, Q6_K 4096 x 14336: 104 us without).
int splits_few(const Weights &w, int tiles) {
    const int64_t groups = (int64_t)tiles * ((w.dim + 127) / 128), want = (768 + groups - 1) / groups, most = w.ffn / 1024;
    return (int)(want < most ? want : most > 1 ? most : 1);
}

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
