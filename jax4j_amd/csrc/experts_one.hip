// One row, or very few (experts.h): the experts of a token or three, in two launches, without an order of pairs and in fp32 throughout.
//
// A call of a few microseconds: what bounds it is what waits for what, and then the stream of W. As in the batch-1 GEMV (gemv_impl.h,
// whose loads and dot products these are) a wave has whole rows of W, a lane the 32 columns of a chunk, so that its loads are
// contiguous kilobytes, and x lies in LDS; the matrix cores, of whose 16 operand rows one row would use one, gain nothing here
// (with them, 8 of 64 Q4_K / Q6_K experts 2048 x 1024: 8.5 and 12.9 us beside the launches around them; this way 9.3 and 8.3, 16.8 a
// call). All weights of a wave are on their way before it waits for x.
//  - experts_one_up: a workgroup has a pair and 16 rows of gate and of up, a wave two of each.
//  - experts_one_down: a wave has a column of a row's result for all slots, its chunks running over slots and ffn; h, times the slot's
//    weight, lies in LDS. No partial results and no further launch.
#include "experts.h"

namespace j4q {
namespace ex {
namespace {

using gemv::f32x2;
using gemv::XChunk;

constexpr int kWaves = 8, kPairs = 2;  // rows of gate and of up a wave

// LDS image of x as gemv_impl.h has it, with a stride of NP chunks: slot j NP + c holds values 4 j .. + 3 of chunk c, behind all of
// them two sums of 16 a chunk. Thread t of T brings values 4 i .. + 3, i = t + T u, into it: every thread of a quad of lanes calls it.
__device__ __forceinline__ void put(f32x4 *xs, float *s16, int NP, int i, int count, f32x4 v) {
    float p = (v.x + v.y) + (v.z + v.w);
    p += gemv::dpp<0xB1>(p);
    p += gemv::dpp<0x4E>(p);
    if (i >= count) return;
    xs[(i & 7) * NP + (i >> 3)] = v;
    if ((i & 3) == 0) s16[i >> 2] = p;
}
__device__ __forceinline__ void get(const f32x4 *xs, const float *s16, int NP, int c, XChunk &x, f32x2 &sums) {
#pragma unroll
    for (int j = 0; j < 8; j++) x.v[j] = xs[j * NP + c];
    sums = reinterpret_cast<const f32x2 *>(s16)[c];
}

// grid: (ffn / 16, pairs). NP >= dim / 32.
template <int FMT, bool HALF, int NP>
__global__ void __launch_bounds__(kWaves * 64)
experts_one_up(Weights w, Call c, float *__restrict__ h) {
    __shared__ f32x4 xs[8 * NP];
    __shared__ __attribute__((aligned(8))) float s16[2 * NP];
    constexpr int XU = (8 * NP + kWaves * 64 - 1) / (kWaves * 64);
    const int t = (int)threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int K = w.dim, N = w.ffn, chunks = K / 32, steps = (chunks + 63) / 64, pair = (int)blockIdx.y;
    // x first: its values come back before the weights'
    const __amdgpu_buffer_rsrc_t xr = make_rsrc((const uint8_t *)c.x + (int64_t)row_of(c, pair) * c.x_stride * (HALF ? 2 : 4), (uint64_t)K * (HALF ? 2u : 4u));
    u32x4 x[XU];
#pragma unroll
    for (int u = 0; u < XU; u++) {
        const uint32_t i = (uint32_t)(t + kWaves * 64 * u);
        if constexpr (HALF) {
            const u32x2 v = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(xr, i < (uint32_t)K / 4u ? 8u * i : kOob, 0, 0));
            x[u] = u32x4{v.x << 16, v.x & 0xFFFF0000u, v.y << 16, v.y & 0xFFFF0000u};
        } else {
            x[u] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(xr, i < (uint32_t)K / 4u ? 16u * i : kOob, 0, 0));
        }
    }
    const int expert = __builtin_amdgcn_readfirstlane(c.ids[pair]);
    if (expert < 0 || expert >= w.experts) return;  // the workgroup as one
    const Rsrc rs[2] = {gemv::rsrc_of(expert_of(w.gate, FMT, expert, N), FMT), gemv::rsrc_of(expert_of(w.up, FMT, expert, N), FMT)};
    Offs ln, rowb, stepb;
    gemv::offsets<FMT>(K, lane, ln, rowb, stepb);
    const uint32_t row0 = blockIdx.x * (uint32_t)(kWaves * kPairs) + (uint32_t)(wave * kPairs);
    Chunk<FMT> set[2][kPairs][2];  // [step parity][row][gate, up]
    auto load = [&](int st, Chunk<FMT> (&s)[kPairs][2]) __attribute__((always_inline)) {
#pragma unroll
        for (int p = 0; p < kPairs; p++) {
            const uint32_t row = row0 + (uint32_t)p, u = (uint32_t)st;
            Offs so = {row * rowb.qs + u * stepb.qs, row * rowb.qh + u * stepb.qh, row * rowb.sc + u * stepb.sc, row * rowb.d + u * stepb.d};
            if (st >= steps) so = Offs{kOob, kOob, kOob, kOob};
            s[p][0].load(rs[0], ln, so);
            s[p][1].load(rs[1], ln, so);
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    load(0, set[0]);
    load(1, set[1]);
#pragma unroll
    for (int u = 0; u < XU; u++) {
        f32x4 v;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const uint32_t b = x[u][j];
            const float f = __builtin_bit_cast(float, b);
            v[j] = fabsf(f) <= 3.402823466e38f ? f : __builtin_nanf("");  // a row that is not finite is NaN as a whole
        }
        put(xs, s16, NP, t + kWaves * 64 * u, K / 4, v);
    }
    __syncthreads();
    float acc[kPairs][2] = {};
    auto process = [&](int st, const Chunk<FMT> (&s)[kPairs][2]) __attribute__((always_inline)) {
        const int at = lane + 64 * st;
        if (at >= chunks) return;
        XChunk xc;
        f32x2 sums;
        get(xs, s16, NP, at, xc, sums);
#pragma unroll
        for (int p = 0; p < kPairs; p++)
#pragma unroll
            for (int m = 0; m < 2; m++) acc[p][m] = s[p][m].apply(xc, sums, acc[p][m], lane & 7);
    };
    for (int st = 0; st < steps; st += 2) {
        process(st, set[0]);
        load(st + 2, set[0]);
        if (st + 1 < steps) process(st + 1, set[1]);
        load(st + 3, set[1]);
    }
#pragma unroll
    for (int p = 0; p < kPairs; p++) {
        const float a = gemv::wave_sum(acc[p][0]), b = gemv::wave_sum(acc[p][1]);
        if (lane == 0) h[(int64_t)pair * N + row0 + p] = activate(a, w.act) * b;
    }
}

// grid: (dim / WAVES, rows). Dynamic LDS: image() bytes; NP = slots * ffn / 32.
template <int FMT, bool HALF, int WAVES>
__global__ void __launch_bounds__(WAVES * 64)
experts_one_down(Weights w, Call c, const float *__restrict__ h, int NP) {
    extern __shared__ f32x4 xs[];
    __shared__ int ids[64];
    float *const s16 = reinterpret_cast<float *>(xs + 8 * NP);
    const int t = (int)threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int K = w.ffn, N = w.dim, per = K / 32, steps = (NP + 63) / 64;
    const int64_t first_pair = (int64_t)blockIdx.y * c.top;
    h += first_pair * K;
    if (t < c.top) ids[t] = c.ids[first_pair + t];
    __syncthreads();
    const Rsrc rs = gemv::rsrc_of(w.down, FMT);
    const Offs rowb = row_bytes<FMT>((uint32_t)K);
    const uint32_t row = blockIdx.x * (uint32_t)WAVES + (uint32_t)wave;
    const Offs so = {row * rowb.qs, row * rowb.qh, row * rowb.sc, row * rowb.d};
    constexpr int D = 4;
    Chunk<FMT> set[D];
    // Step st: chunk j = lane + 64 st, of slot j / per.
    auto load = [&](int st, Chunk<FMT> &s) __attribute__((always_inline)) {
        const int j = lane + 64 * st, slot = j < NP ? j / per : 0, e = j < NP ? ids[slot] : -1;
        const bool ok = e >= 0 && e < w.experts;
        const Offs at = chunk_at<FMT>((uint32_t)(j - slot * per));
        const uint32_t first = (uint32_t)(ok ? e : 0) * (uint32_t)N;
        Offs ln = {first * rowb.qs + at.qs, first * rowb.qh + at.qh, first * rowb.sc + at.sc, first * rowb.d + at.d};
        if (!ok) ln = Offs{kOob, kOob, kOob, kOob};
        s.load(rs, ln, so);
        __builtin_amdgcn_sched_barrier(0);
    };
#pragma unroll
    for (int d = 0; d < D; d++) load(d, set[d]);
    // h times the weights; nothing where there is no expert
    for (int i0 = 0; i0 < 8 * NP; i0 += WAVES * 64) {
        const int i = i0 + t, slot = i < 8 * NP ? i / (K / 4) : 0, e = ids[slot];
        f32x4 v = {};
        if (i < 8 * NP && e >= 0 && e < w.experts) v = reinterpret_cast<const f32x4 *>(h)[i] * c.weights[first_pair + slot];
        put(xs, s16, NP, i, 8 * NP, v);
    }
    __syncthreads();
    float acc = 0.f;
    for (int st = 0; st < steps; st += D) {
#pragma unroll
        for (int d = 0; d < D; d++) {
            const int j = lane + 64 * (st + d);
            if (j < NP) {
                XChunk xc;
                f32x2 sums;
                get(xs, s16, NP, j, xc, sums);
                acc = set[d].apply(xc, sums, acc, lane & 7);
            }
            load(st + d + D, set[d]);
        }
    }
    const float y = gemv::wave_sum(acc);
    if (lane) return;
    const int64_t at = (int64_t)blockIdx.y * c.out_stride + row;
    if constexpr (HALF) ((uint16_t *)c.out)[at] = __builtin_bit_cast(uint16_t, (__bf16)y);
    else ((float *)c.out)[at] = y;
}

constexpr int64_t image(int64_t chunks) { return chunks * (8 * 16 + 8); }

template <int FMT, bool HALF>
hipError_t launch_up(const Weights &w, const Call &c, float *h, hipStream_t s) {
    const dim3 grid((unsigned)(w.ffn / (kWaves * kPairs)), (unsigned)c.pairs);
    if (w.dim <= 2048) experts_one_up<FMT, HALF, 64><<<grid, kWaves * 64, 0, s>>>(w, c, h);
    else if (w.dim <= 4096) experts_one_up<FMT, HALF, 128><<<grid, kWaves * 64, 0, s>>>(w, c, h);
    else experts_one_up<FMT, HALF, 256><<<grid, kWaves * 64, 0, s>>>(w, c, h);
    return hipGetLastError();
}

// 16 waves where the image leaves room for one workgroup a CU alone.
template <int FMT, bool HALF>
hipError_t launch_down(const Weights &w, const Call &c, const float *h, hipEvent_t done, hipStream_t s) {
    const int NP = c.top * (w.ffn / 32), lds = (int)image(NP);
    if (lds > 64 * 1024) {
        if (done) hipExtLaunchKernelGGL((experts_one_down<FMT, HALF, 16>), dim3((unsigned)(w.dim / 16), (unsigned)c.rows), dim3(1024), lds, s, nullptr, done, 0, w, c, h, NP);
        else experts_one_down<FMT, HALF, 16><<<dim3((unsigned)(w.dim / 16), (unsigned)c.rows), 1024, lds, s>>>(w, c, h, NP);
    } else {
        if (done) hipExtLaunchKernelGGL((experts_one_down<FMT, HALF, 8>), dim3((unsigned)(w.dim / 8), (unsigned)c.rows), dim3(512), lds, s, nullptr, done, 0, w, c, h, NP);
        else experts_one_down<FMT, HALF, 8><<<dim3((unsigned)(w.dim / 8), (unsigned)c.rows), 512, lds, s>>>(w, c, h, NP);
    }
    return hipGetLastError();
}

template <int FMT>
hipError_t up_type(const Weights &w, const Call &c, float *h, hipStream_t s) {
    return c.half ? launch_up<FMT, true>(w, c, h, s) : launch_up<FMT, false>(w, c, h, s);
}
template <int FMT>
hipError_t down_type(const Weights &w, const Call &c, const float *h, hipEvent_t done, hipStream_t s) {
    return c.half ? launch_down<FMT, true>(w, c, h, done, s) : launch_down<FMT, false>(w, c, h, done, s);
}

}  // namespace

// The image of all slots' h fits a workgroup's LDS, that of x the kernel.
bool one_fits(const Weights &w, int top) { return w.dim <= 8192 && image((int64_t)top * (w.ffn / 32)) <= 159 * 1024; }

hipError_t launch_one(const Weights &w, const Call &c, hipEvent_t done, hipStream_t s) {
    float *const h = c.part;
    hipError_t e = hipErrorInvalidValue;
    switch (w.up_type) {
    case Q8_0: e = up_type<Q8_0>(w, c, h, s); break;
    case Q4_0: e = up_type<Q4_0>(w, c, h, s); break;
    case Q4_K: e = up_type<Q4_K>(w, c, h, s); break;
    case Q6_K: e = up_type<Q6_K>(w, c, h, s); break;
    }
    if (e != hipSuccess) return e;
    switch (w.down_type) {
    case Q8_0: return down_type<Q8_0>(w, c, h, done, s);
    case Q4_0: return down_type<Q4_0>(w, c, h, done, s);
    case Q4_K: return down_type<Q4_K>(w, c, h, done, s);
    case Q6_K: return down_type<Q6_K>(w, c, h, done, s);
    default: return hipErrorInvalidValue;
    }
}

}  // namespace ex
}  // namespace j4q
