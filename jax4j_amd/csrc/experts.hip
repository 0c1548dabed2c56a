// The experts' products of a layer, host side, and what surrounds the products: the pairs in the order of their experts, x as fp16, the
// weighted sums (experts.h).
#include <limits.h>

#include <algorithm>
#include <exception>
#include <memory>
#include <vector>

#include "arguments.h"
#include "engine.h"
#include "experts.h"
#include "kept_memory.h"
#include "teams.h"

namespace j4q {
namespace ex {
namespace {

constexpr int kMaxExperts = 1024, kMaxTop = 64, kPlanThreads = 512;

// ---- the order of the pairs, and x' -------------------------------------------------------

__device__ __forceinline__ int wave_total(int v) {
#pragma unroll
    for (int o = 32; o > 0; o /= 2) v += __shfl_xor(v, o);
    return v;
}

// Workgroup e < experts: the pairs of expert e in rising order, behind those of the experts before it, and their tiles. Every
// workgroup counts all ids itself, so that none waits for another; each of its waves then places the matches of a contiguous part.
// Bound by the latency of its loads: four ids a lane and load, four loads on their way (32744 pairs of 64 experts 21 us;
// one by one 38).
__device__ void order_pairs(const Weights &w, const Call &c, int e) {
    constexpr int kWaves = kPlanThreads / 64, kStep = 1024;  // ids of a wave and step
    __shared__ int hist[kMaxExperts];
    __shared__ int wave_count[kWaves], sums[3][kWaves];
    const int t = (int)threadIdx.x, lane = t & 63, wave = t >> 6;
    for (int i = t; i < w.experts; i += kPlanThreads) hist[i] = 0;
    __syncthreads();
    const int part = (c.pairs + kWaves * kStep - 1) / (kWaves * kStep) * kStep, from = wave * part, to = from + part < c.pairs ? from + part : c.pairs;
    typedef int32_t i32x4 __attribute__((ext_vector_type(4), aligned(4)));
    // ids i + 256 u + 4 lane .. + 3, u = 0 .. 3; those behind the part's end are no expert's
    auto load = [&](int i, int (&id)[4][4]) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int at = i + 256 * u + 4 * lane;
            if (at + 3 < to) {
                const i32x4 v = *reinterpret_cast<const i32x4 *>(c.ids + at);
#pragma unroll
                for (int j = 0; j < 4; j++) id[u][j] = v[j];
            } else {
#pragma unroll
                for (int j = 0; j < 4; j++) id[u][j] = at + j < to ? c.ids[at + j] : -1;
            }
        }
    };
    int mine = 0;
    for (int i = from; i < to; i += kStep) {
        int id[4][4];
        load(i, id);
#pragma unroll
        for (int u = 0; u < 4; u++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int v = id[u][j];
                if (v >= 0 && v < w.experts) atomicAdd(&hist[v], 1);
                mine += v == e;
            }
    }
    mine = wave_total(mine);
    if (lane == 0) wave_count[wave] = mine;
    __syncthreads();
    int before = 0, up = 0, down = 0;  // pairs and tiles of the experts before this one
    for (int i = t; i < e; i += kPlanThreads) {
        before += hist[i];
        up += (hist[i] + c.up.rows - 1) / c.up.rows;
        down += (hist[i] + c.down.rows - 1) / c.down.rows;
    }
    before = wave_total(before);
    up = wave_total(up);
    down = wave_total(down);
    if (lane == 0) sums[0][wave] = before, sums[1][wave] = up, sums[2][wave] = down;
    __syncthreads();
    before = up = down = 0;
#pragma unroll
    for (int v = 0; v < kWaves; v++) before += sums[0][v], up += sums[1][v], down += sums[2][v];
    const int count = hist[e];
    auto tiles = [&](const Tiles &all, int first) {
        const int own = (count + all.rows - 1) / all.rows;
        // of whole groups of 32 pairs (up to 16: a tile), as even as they can be
        const int per = own && all.rows >= 32 ? ((count + own - 1) / own + 31) / 32 * 32 : all.rows;
        for (int i = t; i < own; i += kPlanThreads) {
            const int left = count - i * per;
            all.tile[first + i] = Tile{e, before + i * per, left < per ? left : per, 0};
        }
        if (e == w.experts - 1 && t == 0) all.count[0] = first + own;
    };
    tiles(c.up, up);
    tiles(c.down, down);
    if (!count) return;
    int at = before;
    for (int v = 0; v < wave; v++) at += wave_count[v];
    if (!wave_count[wave]) return;
    for (int i = from; i < to; i += kStep) {
        int id[4][4];
        load(i, id);
#pragma unroll
        for (int u = 0; u < 4; u++) {
            // matches of the lanes before this one, and of this one's before each of its own
            int own = 0;
#pragma unroll
            for (int j = 0; j < 4; j++) own += id[u][j] == e;
            int ahead = 0, total = 0;
#pragma unroll
            for (int b = 0; b < 3; b++) {  // own is 0 .. 4
                const uint64_t set = __ballot(own >> b & 1);
                ahead += __popcll(set & ((1ull << lane) - 1)) << b;
                total += __popcll(set) << b;
            }
            int place = at + ahead;
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (id[u][j] == e) c.order[place++] = i + 256 * u + 4 * lane + j;
            at += total;
        }
    }
}

// The waves of a team that has a row, so that a lane's values are 4 passes of 8 at most where that can be.
__host__ __device__ inline int row_waves(int K) { return K <= 2048 ? 1 : K <= 4096 ? 2 : K <= 8192 ? 4 : 8; }

// Rows of x as x' in the block layout, their powers and their norms' exponents; 8 / row_waves() of them. Read once, up to 16384
// columns (a workgroup a row, and each read twice: 509 rows of 2048 in fp32 1.5 us more of 175).
__device__ void convert_rows(const Weights &w, const Call &c, int block) {
    __shared__ float most[kPlanThreads / 64], squares[kPlanThreads / 64];
    static_assert(kPlanThreads == 512, "8 waves");
    const int K = w.dim, W = row_waves(K), lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6, t = wave % W * 64 + lane, T = 64 * W;
    const int row = block * (8 / W) + wave / W, chunks = row < c.rows ? K / 8 : 0, r = row < c.rows ? row : 0;
    const uint8_t *const x = (const uint8_t *)c.x + (int64_t)r * c.x_stride * (c.half ? 2 : 4);
    // thread t and pass p: the 8 elements of chunk g = i % 4 of block i / 4, i = t + T p
    auto load = [&](int i, float (&v)[8]) __attribute__((always_inline)) {
        const int at = (i >> 2) * 32 + 4 * (i & 3);
        if (c.half) {
            const u32x2 a = *reinterpret_cast<const u32x2 *>(x + 2 * at), b = *reinterpret_cast<const u32x2 *>(x + 2 * at + 32);
#pragma unroll
            for (int j = 0; j < 2; j++) {
                v[2 * j] = __builtin_bit_cast(float, a[j] << 16);
                v[2 * j + 1] = __builtin_bit_cast(float, a[j] & 0xFFFF0000u);
                v[4 + 2 * j] = __builtin_bit_cast(float, b[j] << 16);
                v[5 + 2 * j] = __builtin_bit_cast(float, b[j] & 0xFFFF0000u);
            }
        } else {
            const f32x4 a = *reinterpret_cast<const f32x4 *>(x + 4 * at), b = *reinterpret_cast<const f32x4 *>(x + 4 * at + 64);
#pragma unroll
            for (int j = 0; j < 4; j++) v[j] = a[j], v[4 + j] = b[j];
        }
    };
    float top = 0.f;
    bool finite = true;
    auto look = [&](const float (&v)[8]) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < 8; j++) {
            top = fmaxf(top, fabsf(v[j]));
            finite &= fabsf(v[j]) <= 3.402823466e38f;
        }
    };
    float held[4][8];
    const bool holds = K <= 2048 * W;
    if (holds) {
#pragma unroll
        for (int p = 0; p < 4; p++)
            if (t + T * p < chunks) load(t + T * p, held[p]);
#pragma unroll
        for (int p = 0; p < 4; p++)
            if (t + T * p < chunks) look(held[p]);
    } else {
        for (int i = t; i < chunks; i += T) {
            float v[8];
            load(i, v);
            look(v);
        }
    }
    top = team_max<64>(finite ? top : __builtin_inff());
    if (W > 1) {
        if (lane == 0) most[wave] = top;
        __syncthreads();
        for (int v = 0; v < W; v++) top = fmaxf(top, most[wave / W * W + v]);
    }
    finite = top <= 3.402823466e38f;
    int e = 0;
    if (finite && top > 0.f) {
        (void)frexpf(top, &e);
        e = 15 - e;
    }
    float sum = 0.f;
    const int64_t lo = (int64_t)c.rows * K;
    _Float16 *const out = c.xa + (int64_t)r * K;
    auto convert = [&](int i, const float (&v)[8]) __attribute__((always_inline)) {
        h8 h, l;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int from = (j & 4) | (j & 1) << 1 | (j >> 1 & 1);  // 0, 2, 1, 3
            const float s = finite ? __builtin_ldexpf(v[from], e) : __builtin_nanf("");
            sum = __builtin_fmaf(s, s, sum);
            h[j] = (_Float16)s;
            l[j] = (_Float16)((s - (float)h[j]) * kLow);
        }
        *reinterpret_cast<h8 *>(out + 8 * i) = h;
        if (!c.half) *reinterpret_cast<h8 *>(out + lo + 8 * i) = l;
    };
    if (holds) {
#pragma unroll
        for (int p = 0; p < 4; p++)
            if (t + T * p < chunks) convert(t + T * p, held[p]);
    } else {
        for (int i = t; i < chunks; i += T) {
            float v[8];
            load(i, v);
            convert(i, v);
        }
    }
    sum = team_sum<64>(sum);
    if (W > 1) {
        if (lane == 0) squares[wave] = sum;
        __syncthreads();
        sum = 0.f;
        for (int v = 0; v < W; v++) sum += squares[wave / W * W + v];
    }
    if (t || !chunks) return;
    int norm = kNothing;
    if (finite && sum > 0.f) {
        (void)frexpf(sum * 1.0001f, &norm);  // above what the sum was rounded by
        norm = ((norm + 1) >> 1) - e;
    }
    c.x_pow[row] = e;
    c.x_norm[row] = finite ? norm : 0;
}

// grid: experts workgroups, and those of the rows.
__global__ void __launch_bounds__(kPlanThreads)
experts_plan(Weights w, Call c) {
    if ((int)blockIdx.x < w.experts) order_pairs(w, c, (int)blockIdx.x);
    else convert_rows(w, c, (int)blockIdx.x - w.experts);
}

// ---- the sums -------------------------------------------------------------------------------

// out[r] = sum over its slots, and each one's splits, one after another, of the weighted partial results. A thread per 4 columns, or 8
// where the partial results are fp16; the loads of 4 slots are on their way together. Memory bounds it: 4093 rows of 2048, 8 slots, 24 us,
// 6.0 TB/s, partly out of the Infinity Cache.
template <bool SMALL>
__global__ void __launch_bounds__(256)
experts_combine(Weights w, Call c) {
    constexpr int V = SMALL ? 8 : 4;
    const int r = (int)(blockIdx.z * gridDim.y + blockIdx.y), col = V * (int)(blockIdx.x * 256 + threadIdx.x);
    if (r >= c.rows || col >= w.dim) return;
    float s[V] = {};
    const int64_t first = (int64_t)r * c.top;
    if constexpr (SMALL) {
        for (int k0 = 0; k0 < c.top; k0 += 4) {
            h8 v[4];
            float weight[4];
            int pow[4];
            bool is[4];
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const int k = k0 + u < c.top ? k0 + u : k0, id = c.ids[first + k];
                is[u] = k0 + u < c.top && id >= 0 && id < w.experts;
                weight[u] = c.weights[first + k];
                pow[u] = 0;
                v[u] = h8{};
                if (is[u]) {
                    pow[u] = c.part_pow[(first + k) * (w.dim / 64) + col / 64];
                    v[u] = *reinterpret_cast<const h8 *>((const _Float16 *)c.part + (first + k) * w.dim + col);
                }
            }
#pragma unroll
            for (int u = 0; u < 4; u++)
                if (is[u]) {
#pragma unroll
                    for (int j = 0; j < V; j++) s[j] += __builtin_ldexpf((float)v[u][j] * weight[u], pow[u]);
                }
        }
    } else {
        for (int k = 0; k < c.top; k++) {
            const int64_t pair = first + k;
            const int id = c.ids[pair];
            if (id < 0 || id >= w.experts) continue;
            for (int v = 0; v < c.splits; v++) {
                const f32x4 p = *reinterpret_cast<const f32x4 *>(c.part + ((int64_t)v * c.pairs + pair) * w.dim + col);
#pragma unroll
                for (int j = 0; j < V; j++) s[j] += p[j];
            }
        }
    }
    if (c.half) {
        typedef __bf16 bf16xv __attribute__((ext_vector_type(V)));
        typedef float f32xv __attribute__((ext_vector_type(V)));
        f32xv t;
#pragma unroll
        for (int j = 0; j < V; j++) t[j] = s[j];
        *reinterpret_cast<bf16xv *>((uint16_t *)c.out + (int64_t)r * c.out_stride + col) = __builtin_convertvector(t, bf16xv);
    } else {
        *reinterpret_cast<f32x4 *>((float *)c.out + (int64_t)r * c.out_stride + col) = f32x4{s[0], s[1], s[2], s[3]};
    }
}

// ---- what is known of the weights -----------------------------------------------------------

// Largest magnitude and sum of squares of a chunk's 32 values. (Squares of weights lie within fp32 by the types alone: |w| < 2^26.)
template <int FMT>
__device__ __forceinline__ void chunk_stats(const Chunk<FMT> &c, int j, float &top, float &sum) {
    uint32_t part[16];
    float s[2], o[2];
    if constexpr (FMT == Q8_0) {
#pragma unroll
        for (int p = 0; p < 8; p++) {
            const uint32_t u = (p < 4 ? c.qa[p & 3] : c.qb[p & 3]) ^ 0x80808080u;
            part[2 * p] = u & 0x00FF00FFu;
            part[2 * p + 1] = u >> 8 & 0x00FF00FFu;
        }
        const float d = half_bits_to_float(c.d);
        s[0] = s[1] = d * 0x1p24f;
        o[0] = o[1] = -128.f * d;
    } else {
#pragma unroll
        for (int p = 0; p < 4; p++) {
            const uint32_t v = c.q[p], t = v >> 8;
            part[2 * p] = v & 0x000F000Fu;
            part[2 * p + 1] = t & 0x000F000Fu;
            part[8 + 2 * p] = v & 0x00F000F0u;
            part[9 + 2 * p] = t & 0x00F000F0u;
            if constexpr (FMT == Q6_K) {
                const uint32_t raw = c.h[p >> 1], hw = p & 1 ? __builtin_amdgcn_alignbit(raw, raw, 8) : raw, u = hw >> 2;
                part[2 * p] |= hw & 0x00300030u;
                part[2 * p + 1] |= u & 0x00300030u;
                part[8 + 2 * p] |= hw & 0x03000300u;
                part[9 + 2 * p] |= u & 0x03000300u;
            }
        }
        if constexpr (FMT == Q4_0) {
            const float d = half_bits_to_float(c.d);
            s[0] = d * 0x1p24f;
            s[1] = d * 0x1p20f;
            o[0] = o[1] = -8.f * d;
        } else if constexpr (FMT == Q4_K) {
            const uint32_t sc = __builtin_amdgcn_ubfe(c.meta.y, 4 * j, 4) | (__builtin_amdgcn_ubfe(c.meta.w, 2 * j, 2) << 4);
            const uint32_t mn = __builtin_amdgcn_ubfe(c.meta.z, 4 * j, 4) | (__builtin_amdgcn_ubfe(c.meta.w, 16 + 2 * j, 2) << 4);
            const float d = half_bits_to_float(c.meta.x & 0xFFFFu) * (float)sc;
            s[0] = d * 0x1p24f;
            s[1] = d * 0x1p20f;
            o[0] = o[1] = -(half_bits_to_float(c.meta.x >> 16) * (float)mn);
        } else {
            const float d = half_bits_to_float(c.d), da = d * (float)(int8_t)(c.s & 0xFFu), db = d * (float)(int8_t)(c.s >> 8 & 0xFFu);
            s[0] = da * 0x1p24f;
            s[1] = db * 0x1p20f;
            o[0] = -32.f * da;
            o[1] = -32.f * db;
        }
    }
    top = sum = 0.f;
#pragma unroll
    for (int p = 0; p < 16; p++) {
        const h2 v = __builtin_bit_cast(h2, part[p]);
        const float a = __builtin_fmaf((float)v.x, s[p >> 3], o[p >> 3]), b = __builtin_fmaf((float)v.y, s[p >> 3], o[p >> 3]);
        top = fmaxf(top, fmaxf(fabsf(a), fabsf(b)));
        sum = __builtin_fmaf(a, a, __builtin_fmaf(b, b, sum));
    }
}

// Of every row of a matrix of `experts` x rows: max |w| 2^pow in [2^13, 2^14) and the exponent of the norm (NULL: not asked for). A wave per
// row, straight from the codes: what it reads is what bounds it. grid: (rows / 4, experts).
template <int FMT>
__global__ void __launch_bounds__(256)
row_stats(QMat all, int rows, int32_t *__restrict__ pow, int32_t *__restrict__ norm) {
    const int lane = (int)threadIdx.x & 63, row = __builtin_amdgcn_readfirstlane(4 * (int)blockIdx.x + ((int)threadIdx.x >> 6)), expert = (int)blockIdx.y;
    if (row >= rows) return;
    const Rsrc r = gemv::rsrc_of(expert_of(all, FMT, expert, rows), FMT);
    const uint32_t K = (uint32_t)all.cols;
    const Offs rb = row_bytes<FMT>(K), so{rb.qs * (uint32_t)row, rb.qh * (uint32_t)row, rb.sc * (uint32_t)row, rb.d * (uint32_t)row};
    float top = 0.f;
    double sum = 0.;
    for (uint32_t c = (uint32_t)lane; c < K / 32; c += 64) {
        Chunk<FMT> v;
        v.load(r, chunk_at<FMT>(c), so);
        float t, q;
        chunk_stats<FMT>(v, (int)(c & 7), t, q);
        top = fmaxf(top, t);
        sum += (double)q;
    }
#pragma unroll
    for (int o = 32; o > 0; o /= 2) {
        top = fmaxf(top, __shfl_xor(top, o));
        sum += __shfl_xor(sum, o);
    }
    if (lane) return;
    int p = 0, q = kNothing;
    if (top > 0.f && top <= 3.402823466e38f) {
        (void)frexpf(top, &p);
        p = 14 - p;
    }
    if (sum > 0.) {
        if (sum < 1e300) {
            (void)frexp(sum * 1.0001, &q);
            q = (q + 1) >> 1;
        } else {  // weights that are not finite: what they reach is not either
            q = 0;
        }
    }
    pow[(int64_t)expert * rows + row] = p;
    if (norm) norm[(int64_t)expert * rows + row] = q;
}

// bound[e] = the largest sum of the exponents of a gate row of expert e (of `rows`) and of the same up row.
__global__ void __launch_bounds__(256)
expert_bound(const int32_t *__restrict__ gate, const int32_t *__restrict__ up, int rows, int32_t *__restrict__ bound) {
    __shared__ int most[4];
    const int t = (int)threadIdx.x;
    const int64_t first = (int64_t)blockIdx.x * rows;
    int a = 2 * kNothing;
    for (int i = t; i < rows; i += 256) {
        const int v = gate[first + i] + up[first + i];
        a = a > v ? a : v;
    }
#pragma unroll
    for (int o = 32; o > 0; o /= 2) {
        const int v = __shfl_xor(a, o);
        a = a > v ? a : v;
    }
    if ((t & 63) == 0) most[t >> 6] = a;
    __syncthreads();
    if (t) return;
    for (int v = 1; v < 4; v++) a = a > most[v] ? a : most[v];
    bound[blockIdx.x] = a;
}

// ---- handles --------------------------------------------------------------------------------

struct Experts {
    j4q_experts_config c{};
    uint32_t gen = 0;
    bool live = false;
    Weights w{};
    uint64_t weight_bytes = 0, bytes = 0;
    void *dev = nullptr;
};

std::vector<std::unique_ptr<Experts>> g_experts;

Experts *lookup(j4q_experts h) {
    const uint64_t lo = h & 0xffffffffu;
    if (lo == 0 || lo > g_experts.size()) return nullptr;
    Experts *k = g_experts[lo - 1].get();
    return k->live && k->gen == (uint32_t)(h >> 32) ? k : nullptr;
}

int get(j4q_experts h, const char *op, Experts **out) {
    *out = lookup(h);
    return *out ? J4Q_OK : report_error(J4Q_EHANDLE, "%s: unknown or destroyed experts 0x%llx", op, (unsigned long long)h);
}

int no_memory(const char *op) { return report_error(J4Q_ENOMEM, "%s failed: out of host memory", op); }

bool type_ok(int type, int64_t cols) {
    switch (type) {
    case Q8_0: return cols % 64 == 0;
    case Q4_0: return cols % 128 == 0;
    case Q4_K:
    case Q6_K: return cols % 256 == 0;
    default: return false;
    }
}

// The powers of a matrix's rows and, but for NULL, the exponents of their norms, `rows` of each expert.
hipError_t stats(int type, const QMat &m, int experts, int rows, int32_t *pow, int32_t *norm, hipStream_t s) {
    const dim3 grid((unsigned)((rows + 3) / 4), (unsigned)experts);
    switch (type) {
    case Q8_0: row_stats<Q8_0><<<grid, 256, 0, s>>>(m, rows, pow, norm); break;
    case Q4_0: row_stats<Q4_0><<<grid, 256, 0, s>>>(m, rows, pow, norm); break;
    case Q4_K: row_stats<Q4_K><<<grid, 256, 0, s>>>(m, rows, pow, norm); break;
    case Q6_K: row_stats<Q6_K><<<grid, 256, 0, s>>>(m, rows, pow, norm); break;
    default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

int create(const j4q_experts_config &c, j4q_experts *out) {
    abi::QuantRef gate, up, down;
    int rc;
    if ((rc = abi::quant_locked(c.gate, "experts", &gate)) || (rc = abi::quant_locked(c.up, "experts", &up)) || (rc = abi::quant_locked(c.down, "experts", &down)))
        return rc;
    const int64_t E = c.experts, dim = gate.cols, ffn = down.cols;
    if (gate.qtype != up.qtype || gate.rows != up.rows || gate.cols != up.cols)
        return report_error(J4Q_EINVAL, "experts: gate is type %d [%lld, %lld], up type %d [%lld, %lld]", gate.qtype, (long long)gate.rows, (long long)gate.cols,
                            up.qtype, (long long)up.rows, (long long)up.cols);
    if (gate.rows != E * ffn || down.rows != E * dim)
        return report_error(J4Q_EINVAL, "experts: %lld experts with gate and up [%lld, %lld], down [%lld, %lld]", (long long)E, (long long)gate.rows,
                            (long long)gate.cols, (long long)down.rows, (long long)down.cols);
    if (!type_ok(gate.qtype, dim) || !type_ok(down.qtype, ffn) || dim > 65536 || ffn > 65536)
        return report_error(J4Q_EUNSUPPORTED, "experts: type %d of %lld columns, type %d of %lld (Q8_0, a multiple of 64 columns, Q4_0, of 128, Q4_K, Q6_K; at most 65536)",
                            gate.qtype, (long long)dim, down.qtype, (long long)ffn);
    if (dim * ffn >= 1ll << 31) return report_error(J4Q_EUNSUPPORTED, "experts: matrices of %lld x %lld values (fewer than 2^31)", (long long)dim, (long long)ffn);
    if ((rc = abi::ready_locked())) return rc;
    if (capturing(abi::stream())) return report_error(J4Q_EINVAL, "experts: the engine stream is captured");
    size_t slot = 0;
    while (slot < g_experts.size() && g_experts[slot]->live) slot++;
    if (slot == g_experts.size()) g_experts.emplace_back(new Experts);
    Experts &k = *g_experts[slot];
    const uint64_t words = (uint64_t)(4 * E * ffn + 2 * E * dim + 2 * E);  // bounds; powers and norms of gate and up; powers of down (E dim and E words are to spare)
    void *dev = nullptr;
    hipError_t e = abi::malloc_locked(&dev, words * 4);
    if (e != hipSuccess) return report_hip("experts", e);
    const hipStream_t s = abi::stream();
    int32_t *const at = (int32_t *)dev;
    k.w = Weights{};
    k.w.gate = gate.m;
    k.w.up = up.m;
    k.w.down = down.m;
    k.w.up_type = gate.qtype;
    k.w.down_type = down.qtype;
    k.w.experts = (int)E;
    k.w.dim = (int)dim;
    k.w.ffn = (int)ffn;
    k.w.act = c.activation;
    int32_t *const gate_pow = at + 2 * E, *const up_pow = gate_pow + E * ffn, *const gate_norm = up_pow + E * ffn, *const up_norm = gate_norm + E * ffn,
                  *const down_pow = up_norm + E * ffn;
    k.w.bound = at;
    k.w.gate_pow = gate_pow;
    k.w.up_pow = up_pow;
    k.w.down_pow = down_pow;
    e = stats(gate.qtype, gate.m, (int)E, (int)ffn, gate_pow, gate_norm, s);
    if (e == hipSuccess) e = stats(up.qtype, up.m, (int)E, (int)ffn, up_pow, up_norm, s);
    if (e == hipSuccess) e = stats(down.qtype, down.m, (int)E, (int)dim, down_pow, nullptr, s);
    if (e == hipSuccess) {
        expert_bound<<<(unsigned)E, 256, 0, s>>>(gate_norm, up_norm, (int)ffn, at);
        e = hipGetLastError();
    }
    if (e == hipSuccess) e = hipStreamSynchronize(s);
    if (e != hipSuccess) {
        (void)hipFree(dev);
        return report_hip("experts", e);
    }
    k.c = c;
    k.dev = dev;
    k.bytes = words * 4;
    k.weight_bytes = gate.gguf_bytes + up.gguf_bytes + down.gguf_bytes;
    k.gen++;
    k.live = true;
    const j4q_experts h = (uint64_t)k.gen << 32 | (uint64_t)(slot + 1);
    for (j4q_buffer b : {c.gate, c.up, c.down}) (void)abi::pin_locked(b, h);
    *out = h;
    return J4Q_OK;
}

// The parts of a call's workspace; bytes in all.
uint64_t lay_out(const Weights &w, Call *c, uint8_t *base) {
    uint64_t at = 0;
    auto take = [&](uint64_t n) {
        uint8_t *const p = base + at;
        at += align256(n);
        return p;
    };
    if (c->one) {
        c->part = (float *)take(4 * (uint64_t)c->pairs * (uint64_t)w.ffn);
        return at;
    }
    const uint64_t planes = c->half ? 1 : 2, P = (uint64_t)c->pairs, T = (uint64_t)c->rows;
    c->up.count = (int32_t *)take(8);
    c->down.count = c->up.count + 1;
    c->order = (int32_t *)take(4 * P);
    c->up.tile = (Tile *)take(sizeof(Tile) * (uint64_t)c->up.most);
    c->down.tile = (Tile *)take(sizeof(Tile) * (uint64_t)c->down.most);
    c->x_pow = (int32_t *)take(4 * T);
    c->x_norm = (int32_t *)take(4 * T);
    c->xa = (_Float16 *)take(2 * planes * T * (uint64_t)w.dim);
    c->ha = (_Float16 *)take(2 * planes * P * (uint64_t)w.ffn);
    c->part = (float *)take((c->small ? 2 : 4 * (uint64_t)c->splits) * P * (uint64_t)w.dim);
    c->part_pow = (int32_t *)take(c->small ? 4 * P * (uint64_t)(w.dim / 64) : 0);
    return at;
}

// Rows of a tile, and how many tiles a call has at most.
void shape(const Weights &w, Call *c) {
    // A row, or up to three with so few pairs that hardly two share an expert: two launches rather than four (3 rows, 4 of 32 experts 1024 x
    // 512: 24.1 -> 13.9 us; 2, 2 of 8 of 4096 x 14336: 118 -> 109), which read an expert's weights for each of its pairs (4, 8 of 64: 44.5 -> 46.8).
    c->one = (c->rows == 1 || (c->rows <= 3 && 2 * c->pairs <= w.experts)) && one_fits(w, c->top);
    const int each = c->pairs / w.experts, some = w.experts < c->pairs ? w.experts : c->pairs, few = c->half ? 16 : 8;
    c->few = each < 24;  // (4 of 32 experts 2048 x 1024, bf16, 22 pairs each: tiles of 16 78.6 us, of 32 82; 30 each: 92, 82)
    c->up.rows = c->few ? few : rows_many(w.up_type, c->half, each);
    c->down.rows = c->few ? few : rows_many(w.down_type, c->half, each);
    for (Tiles *t : {&c->up, &c->down}) t->most = some + (c->pairs - some) / t->rows;
    c->splits = c->few ? splits_few(w, c->down.most) : 1;
    c->small = c->half && !c->few;
}

int check_size(const char *op, int64_t rows, int32_t top, int type) {
    if (!dense_type(type)) return report_error(J4Q_EUNSUPPORTED, "%s: type %d (J4Q_KIND_F32 or J4Q_KIND_BF16)", op, type);
    if (rows < 1 || top < 1 || top > kMaxTop) return report_error(J4Q_EINVAL, "%s: %lld rows of %d experts (1 to %d)", op, (long long)rows, top, kMaxTop);
    if (rows > (1 << 22) / top) return report_error(J4Q_EUNSUPPORTED, "%s: %lld rows of %d experts (at most %d pairs)", op, (long long)rows, top, 1 << 22);
    return J4Q_OK;
}

hipError_t launch(const Weights &w, const Call &c, hipEvent_t done, hipStream_t s) {
    if (c.one) return launch_one(w, c, done, s);
    const int rows = 8 / row_waves(w.dim);
    experts_plan<<<(unsigned)(w.experts + (c.rows + rows - 1) / rows), kPlanThreads, 0, s>>>(w, c);
    hipError_t e = hipGetLastError();
    const auto products = c.few ? launch_few : launch_many;
    if (e == hipSuccess) e = products(w, c, false, s);
    if (e == hipSuccess) e = products(w, c, true, s);
    if (e != hipSuccess) return e;
    const int y = c.rows < 32768 ? c.rows : 32768;
    const int cols = c.small ? 2048 : 1024;
    const dim3 grid((unsigned)((w.dim + cols - 1) / cols), (unsigned)y, (unsigned)((c.rows + y - 1) / y));
    return c.small ? launch_with_event(experts_combine<true>, grid, dim3(256), s, done, w, c) : launch_with_event(experts_combine<false>, grid, dim3(256), s, done, w, c);
}

// A call of many rows runs as ranges of rows, one after another in the same workspace: the products address x' and h' by 32-bit offsets,
// and what a range of 2^17 pairs needs (2 GiB of results at dim 4096, fp32) is enough for whole tiles of 1024 experts.
struct Ranges {
    int count, rows, larger;  // `larger` ranges of rows + 1 and then count - larger of rows
};

Ranges ranges(const Weights &w, const Call &c) {
    const int64_t bytes = c.half ? 2 : 4, limit = (1ll << 31) - 1;
    int64_t most = (1 << 17) / c.top;
    most = std::min(most, limit / (bytes * w.dim));
    most = std::min(most, limit / (bytes * w.ffn * c.top));
    const int n = (int)((c.rows + most - 1) / most);
    return {n, c.rows / n, c.rows % n};
}

Call range(const Weights &w, const Call &all, int first, int rows) {
    Call c = all;
    const int64_t e = c.half ? 2 : 4;
    c.x = (const uint8_t *)all.x + first * all.x_stride * e;
    c.out = (uint8_t *)all.out + first * all.out_stride * e;
    c.ids = all.ids + (int64_t)first * c.top;
    c.weights = all.weights + (int64_t)first * c.top;
    c.rows = rows;
    c.pairs = rows * c.top;
    c.top_inverse = (uint32_t)(((1ull << 32) + (uint64_t)c.top - 1) / (uint64_t)c.top);
    shape(w, &c);
    return c;
}

uint64_t workspace(const Weights &w, const Call &all) {
    const Ranges r = ranges(w, all);
    uint64_t most = 0;
    for (int more = 0; more < 2; more++) {
        if (!(more ? r.larger : r.count - r.larger)) continue;
        Call c = range(w, all, 0, r.rows + more);
        most = std::max(most, lay_out(w, &c, nullptr));
    }
    return most;
}

hipError_t launch_all(const Weights &w, const Call &all, void *space, hipEvent_t done, hipStream_t s) {
    const Ranges r = ranges(w, all);
    hipError_t e = hipSuccess;
    for (int i = 0, first = 0; i < r.count && e == hipSuccess; i++) {
        Call c = range(w, all, first, r.rows + (i < r.larger));
        lay_out(w, &c, (uint8_t *)space);
        e = launch(w, c, i + 1 == r.count ? done : nullptr, s);
        first += c.rows;
    }
    return e;
}

int apply(const Experts &k, const j4q_experts_args &a, hipStream_t s) {
    Call c{};
    c.x = a.x;
    c.x_stride = a.x_stride ? a.x_stride : k.w.dim;
    c.ids = a.ids;
    c.weights = a.weights;
    c.out = a.out;
    c.out_stride = a.out_stride ? a.out_stride : k.w.dim;
    c.rows = (int)a.rows;
    c.top = a.top_k;
    c.half = a.type == J4Q_KIND_BF16;
    const int64_t e = dense_size(a.type), dim = k.w.dim;
    for (int64_t st : {c.x_stride, c.out_stride})
        if (st < dim || st > 1ll << 36 || st * e % 16) return report_error(J4Q_EINVAL, "experts apply: rows of %lld values %lld apart, a multiple of 16 bytes", (long long)dim, (long long)st);
    if (!aligned(a.x, 16) || !aligned(a.out, 16) || !aligned(a.ids, 4) || !aligned(a.weights, 4))
        return report_error(J4Q_EINVAL, "experts apply: x and out must be 16-byte aligned, ids and weights 4-byte aligned");
    const uint64_t out_bytes = (uint64_t)(((c.rows - 1) * c.out_stride + dim) * e), x_bytes = (uint64_t)(((c.rows - 1) * c.x_stride + dim) * e),
                   pair_bytes = (uint64_t)c.rows * (uint64_t)c.top * 4;
    if (overlap(c.x, c.x_stride * e, dim * e, c.out, c.out_stride * e, dim * e, c.rows) || overlap(c.ids, pair_bytes, c.out, out_bytes) ||
        overlap(c.weights, pair_bytes, c.out, out_bytes))
        return report_error(J4Q_EUNSUPPORTED, "experts apply: out must lie apart from x, ids and weights");
    const uint64_t bytes = workspace(k.w, c);
    if (a.workspace) {
        if (!aligned(a.workspace, 256) || a.workspace_bytes < bytes)
            return report_error(J4Q_EINVAL, "experts apply: a workspace of %llu bytes, 256-byte aligned, is needed", (unsigned long long)bytes);
        if (overlap(a.workspace, bytes, c.x, x_bytes) || overlap(a.workspace, bytes, c.out, out_bytes) || overlap(a.workspace, bytes, c.ids, pair_bytes) ||
            overlap(a.workspace, bytes, c.weights, pair_bytes))
            return report_error(J4Q_EUNSUPPORTED, "experts apply: the workspace must lie apart from the other arguments");
    }
    int rc;
    if ((rc = abi::ready_locked())) return rc;
    if (!s) s = abi::stream();
    if (a.workspace) {
        const hipError_t err = launch_all(k.w, c, a.workspace, nullptr, s);
        return err == hipSuccess ? J4Q_OK : report_hip("experts apply", err);
    }
    Workspace ws;
    hipError_t err = abi::workspace_begin_locked(s, bytes, &ws);
    if (err != hipSuccess) return report_hip("experts apply", err);
    err = launch_all(k.w, c, ws.ptr, ws.done, s);
    abi::workspace_end_locked(s, ws, err == hipSuccess);
    return err == hipSuccess ? J4Q_OK : report_hip("experts apply", err);
}

}  // namespace
}  // namespace ex
}  // namespace j4q

using namespace j4q;

extern "C" {

int j4q_experts_create(const j4q_experts_config *config, j4q_experts *out) try {
    if (!config || !out) return report_error(J4Q_EINVAL, "experts: NULL argument");
    if (config->experts < 1 || config->experts > ex::kMaxExperts) return report_error(J4Q_EINVAL, "experts: %d of them (1 to %d)", config->experts, ex::kMaxExperts);
    if (config->activation < J4Q_ACT_SILU || config->activation > J4Q_ACT_RELU) return report_error(J4Q_EUNSUPPORTED, "experts: unknown activation %d", config->activation);
    std::lock_guard<std::mutex> lk(abi::lock());
    return ex::create(*config, out);
} catch (const std::exception &) {
    return ex::no_memory("experts");
}

int j4q_experts_destroy(j4q_experts h) {
    if (h == 0) return J4Q_OK;
    std::lock_guard<std::mutex> lk(abi::lock());
    ex::Experts *k;
    int rc;
    if ((rc = ex::get(h, "experts destroy", &k)) || (rc = abi::ready_locked())) return rc;
    const hipError_t e = hipDeviceSynchronize();
    if (e != hipSuccess) return report_hip("experts destroy", e);
    (void)hipFree(k->dev);
    for (j4q_buffer b : {k->c.gate, k->c.up, k->c.down}) abi::unpin_locked(b);
    k->dev = nullptr;
    k->live = false;
    return J4Q_OK;
}

int j4q_experts_info(j4q_experts h, j4q_experts_desc *out) {
    if (!out) return report_error(J4Q_EINVAL, "experts info: NULL argument");
    std::lock_guard<std::mutex> lk(abi::lock());
    ex::Experts *k;
    const int rc = ex::get(h, "experts info", &k);
    if (rc) return rc;
    *out = j4q_experts_desc{k->c, k->w.dim, k->w.ffn, k->weight_bytes, k->bytes};
    return J4Q_OK;
}

int j4q_experts_workspace(j4q_experts h, int64_t rows, int32_t top_k, int type, uint64_t *bytes) {
    if (!bytes) return report_error(J4Q_EINVAL, "experts workspace: NULL argument");
    std::lock_guard<std::mutex> lk(abi::lock());
    ex::Experts *k;
    int rc;
    if ((rc = ex::get(h, "experts workspace", &k)) || (rc = ex::check_size("experts workspace", rows, top_k, type))) return rc;
    ex::Call c{};
    c.rows = (int)rows;
    c.top = top_k;
    c.half = type == J4Q_KIND_BF16;
    *bytes = ex::workspace(k->w, c);
    return J4Q_OK;
}

int j4q_experts_apply(j4q_experts h, const j4q_experts_args *args, void *stream) {
    if (!args || !args->x || !args->ids || !args->weights || !args->out) return report_error(J4Q_EINVAL, "experts apply: NULL argument");
    std::lock_guard<std::mutex> lk(abi::lock());
    ex::Experts *k;
    int rc;
    if ((rc = ex::get(h, "experts apply", &k)) || (rc = ex::check_size("experts apply", args->rows, args->top_k, args->type))) return rc;
    return ex::apply(*k, *args, (hipStream_t)stream);
}

}  // extern "C"
