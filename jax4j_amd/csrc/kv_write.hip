// What writes the 8-bit key/value cache and reads it back: rotary positions, append (rotate, quantize, store), read
// (dequantize), copies of pages, and the small updates of tables on the device. All are bound by memory or, at a step of one
// token, by their launch.
//
// Rotary positions turn pair (u, w) of a row by the angle whose cosine c and sine s the caller's tables hold:
// u' = u c - w s, w' = w c + u s, each product rounded to fp32 before the sum (no fma), so that a key's codes are those of
// the same formula in any program.
// A block of 16 tokens x D of a head has one scale for its keys and one for its values. Where the new tokens begin the block
// it is max(amax / 127, 2^-64); else the scale that is there, times the least power of two under which
// every code fits 8 bits: the codes that are there are then divided by that power, which rounds them once more per
// doubling, so that the error of a code stays below one step of the final scale (a half, and a quarter, an eighth.. before).
// A block of zeros (its scale the least one) gets amax / 127 as one without tokens does.
// A value that is not finite makes the whole block of its head NaN: the cache has no code for it, and NaN is not lost.
// Measured at: append, below; read 24 MB of codes to fp32 (245 MB in all) 47 us, 5.1 TB/s; copies of 256 pages of 131 KB in 4
// layers (269 MB) 41 to 47 us; a step's tables 2 us.
#include "kv.h"

#include <float.h>

#include <algorithm>

namespace j4q {
namespace {

__device__ __forceinline__ float bf16_at(const void *p, int64_t i) {
    return __builtin_bit_cast(float, (uint32_t)((const uint16_t *)p)[i] << 16);
}
__device__ __forceinline__ uint16_t to_bf16(float f) {
    const uint32_t u = __builtin_bit_cast(uint32_t, f);
    if ((u & 0x7fffffffu) > 0x7f800000u) return (uint16_t)((u >> 16) | 0x40);
    return (uint16_t)((u + 0x7fffu + ((u >> 16) & 1)) >> 16);
}

// The sequence i of n with first[i] <= at < first[i + 1].
__device__ __forceinline__ int sequence_of(const int32_t *first, int n, int at) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (first[mid] <= at) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// Cosine and sine of pair `pair` of row `row`, which is token `place` of its sequence.
__device__ __forceinline__ float2 turn_of(const KvRope &r, int pair, int64_t row, int place) {
    const int at = r.positions ? r.positions[(r.axes > 1 ? (int64_t)r.axis[pair] * r.rows : 0) + row] : place;
    if (at < 0 || at >= r.table_rows) return make_float2(__builtin_nanf(""), __builtin_nanf(""));  // no angle in the tables
    const int64_t i = (int64_t)at * r.pairs + pair;
    return make_float2(r.cos[i], r.sin[i]);
}
__device__ __forceinline__ void turn(float c, float s, float &u, float &w) {
#pragma clang fp contract(off)
    const float uc = u * c, ws = w * s, wc = w * c, us = u * s;
    u = uc - ws;
    w = wc + us;
}

// V consecutive values, 4 of them or 8 bf16 in pieces of 16 (or 8) bytes.
template <int V>
__device__ __forceinline__ void load(const void *p, int64_t i, bool bf16, float *x) {
    if constexpr (V == 1) {
        x[0] = bf16 ? bf16_at(p, i) : ((const float *)p)[i];
    } else if (bf16) {
        uint32_t w[V / 2];
        if constexpr (V == 8) *(uint4 *)w = *(const uint4 *)((const uint16_t *)p + i);
        else *(uint2 *)w = *(const uint2 *)((const uint16_t *)p + i);
#pragma unroll
        for (int j = 0; j < V / 2; j++) {
            x[2 * j] = __builtin_bit_cast(float, w[j] << 16);
            x[2 * j + 1] = __builtin_bit_cast(float, w[j] & 0xffff0000u);
        }
    } else {
#pragma unroll
        for (int j = 0; j < V; j += 4) *(float4 *)(x + j) = *(const float4 *)((const float *)p + i + j);
    }
}
template <int V>
__device__ __forceinline__ void store(void *p, int64_t i, bool bf16, const float *x) {
    if constexpr (V == 1) {
        if (bf16) ((uint16_t *)p)[i] = to_bf16(x[0]);
        else ((float *)p)[i] = x[0];
    } else if (bf16) {
        uint32_t w[V / 2];
#pragma unroll
        for (int j = 0; j < V / 2; j++) w[j] = to_bf16(x[2 * j]) | (uint32_t)to_bf16(x[2 * j + 1]) << 16;
        if constexpr (V == 8) *(uint4 *)((uint16_t *)p + i) = *(const uint4 *)w;
        else *(uint2 *)((uint16_t *)p + i) = *(const uint2 *)w;
    } else {
#pragma unroll
        for (int j = 0; j < V; j += 4) *(float4 *)((float *)p + i + j) = *(const float4 *)(x + j);
    }
}

// A workgroup turns heads [head0, head0 + heads) of rows [row0, row0 + rows). An item is 2 V channels of a head: V pairs that are
// turned, or channels behind those, which are copied. The rows' cosines and sines are looked up once, into LDS, whatever the number
// of heads (looked up by every item they were three times as many loads as the values), while the items' values are on
// their way. In place is fine: a thread reads what it writes.
constexpr int kRopePairs = 1024;  // of a workgroup's rows together
// Items of a thread: a head in single pairs is one workgroup's; else two, which leave registers for 6 workgroups a CU and more.
constexpr int rope_items(int v) { return v == 1 ? 4 : 2; }
static_assert(256 * rope_items(1) >= kRopeMaxDim / 2 && 256 * rope_items(4) >= 512 && 256 * rope_items(8) >= 512, "");  // see rope_grid
struct RopeRows {
    const void *x;
    void *out;
    int64_t stride, out_stride;  // of the rows
    int32_t dim, bf16;
};
template <int V>
__device__ __forceinline__ void rope_rows(const RopeRows &g, const KvRope &r, int64_t row0, int rows, int head0, int heads, const KvStep *step,
                                          float2 *angles) {
    constexpr int kRopeItems = rope_items(V);
    const int units = g.dim / (2 * V), per_row = units * heads, count = rows * per_row;
    float a[kRopeItems][2][V];
    int row[kRopeItems], unit[kRopeItems], at0[kRopeItems], at1[kRopeItems];
    int64_t head_at[kRopeItems];
#pragma unroll
    for (int j = 0; j < kRopeItems; j++) {
        const int item = min((int)threadIdx.x + 256 * j, count - 1);
        row[j] = item / per_row;
        const int rest = item - row[j] * per_row, head = rest / units;
        unit[j] = rest - head * units;
        head_at[j] = (int64_t)(head0 + head) * g.dim;
        const int i = unit[j] * V;
        const bool halves = i < r.pairs && !r.interleaved;
        at0[j] = halves ? i : 2 * i;
        at1[j] = halves ? i + r.pairs : 2 * i + V;
        if ((int)threadIdx.x + 256 * j < count) {
            const int64_t from = (row0 + row[j]) * g.stride + head_at[j];
            load<V>(g.x, from + at0[j], g.bf16, a[j][0]);
            load<V>(g.x, from + at1[j], g.bf16, a[j][1]);
        }
    }
    if (r.pairs)
        for (int t = threadIdx.x; t < rows * r.pairs; t += 256) {
            const int k = t / r.pairs;
            int place = 0;
            if (step && !r.positions) {
                const int at = (int)row0 + k, i = step->rows == step->n ? at : sequence_of(step->row0, step->n, at);  // a token each: no search
                place = step->len[i] - step->row0[i + 1] + (int)row0 + k;
            }
            angles[t] = turn_of(r, t - k * r.pairs, row0 + k, place);
        }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kRopeItems; j++) {
        if ((int)threadIdx.x + 256 * j >= count) break;
        const int i = unit[j] * V;
        if (i < r.pairs) {
            float *f = &a[j][0][0];
            const float2 *cs = angles + row[j] * r.pairs + i;
            if (r.interleaved) {
#pragma unroll
                for (int e = 0; e < V; e++) turn(cs[e].x, cs[e].y, f[2 * e], f[2 * e + 1]);
            } else {
#pragma unroll
                for (int e = 0; e < V; e++) turn(cs[e].x, cs[e].y, f[e], f[V + e]);
            }
        }
        const int64_t to = (row0 + row[j]) * g.out_stride + head_at[j];
        store<V>(g.out, to + at0[j], g.bf16, a[j][0]);
        store<V>(g.out, to + at1[j], g.bf16, a[j][1]);
    }
}

// Rows and heads of a workgroup: about 512 items where there are enough of them (video patches of 16381 x 16 heads of 80 in bf16: 21.6
// us, with 1024 26.7 and with 256 26.6), else 256.
struct RopeGrid {
    int rows, heads;
    int64_t groups_x, groups_y;  // over rows, over heads
};
RopeGrid rope_grid(int64_t rows, int heads, int dim, int v, int pairs) {
    const int units = dim / (2 * v);
    const int64_t items = rows * heads * units;
    const int want = items >= 512 * 1024 ? 512 : 256;
    RopeGrid g;
    g.heads = std::max(1, std::min(heads, std::max(want, units) / units));
    g.rows = (int)std::max<int64_t>(1, std::min<int64_t>({rows, want / (units * g.heads), pairs ? kRopePairs / pairs : 1024}));
    g.groups_x = (rows + g.rows - 1) / g.rows;
    g.groups_y = (heads + g.heads - 1) / g.heads;
    return g;
}

template <int V>
__global__ void __launch_bounds__(256) rope_kernel(RopeRows g, int64_t rows, int heads, int rows_each, int heads_each, KvRope r) {
    __shared__ float2 angles[kRopePairs];
    const int64_t row0 = (int64_t)blockIdx.x * rows_each;
    const int head0 = blockIdx.y * heads_each;
    rope_rows<V>(g, r, row0, (int)min((int64_t)rows_each, rows - row0), head0, min(heads_each, heads - head0), nullptr, angles);
}

__device__ __forceinline__ float block_max(float v, float *red) {
    for (int d = 32; d; d >>= 1) v = fmaxf(v, __shfl_xor(v, d));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
}

// The block's scale after values of magnitude up to amax, and what the codes that are there are multiplied by.
__device__ __forceinline__ float next_scale(float amax, bool begun, float old, float *shrink) {
    *shrink = 1.0f;
    if (!(amax <= FLT_MAX)) return __builtin_nanf("");
    if (begun && old != old) return old;
    if (!begun || old <= kKvMinScale) {
        const float s = fmaxf(amax / 127.0f, kKvMinScale);
        if (begun) *shrink = old / s;
        return s;
    }
    const float r = 1.0f / old;
    float a = amax;
    while (a * r >= 127.5f) {
        a *= 0.5f;
        old *= 2.0f;
        *shrink *= 0.5f;
    }
    return old;
}
__device__ __forceinline__ uint32_t code_of(float x, float r) { return (uint32_t)(int)rintf(x * r) & 0xffu; }
__device__ __forceinline__ uint32_t shrink_of(uint32_t code, float f) { return (uint32_t)(int)rintf((float)(int8_t)code * f) & 0xffu; }

// One block of 16 tokens of a kv head per workgroup, 256 threads; the workgroups behind them, whose work is shorter, turn the
// queries. A step of one token is bound by its chain of loads, so what does not need another load's answer goes with it:
// values and the page, then scales, codes that are there and angles (64 sequences of a token, 8 kv heads of 128 and 32 query
// heads: 6.5 us, and 5.9 so). A prompt is bound by memory: 16384 blocks 66 us, 5.0 TB/s (one load after the other 98); 2043
// tokens with their queries 22.2 us, 4.0 TB/s.
template <int D>
__global__ void __launch_bounds__(256) append_kernel(KvAppend a) {
    constexpr int P = D + 4;
    __shared__ __align__(16) float xs[2][kKvBlock][P];
    __shared__ float red[2][4];
    const int tid = threadIdx.x;
    const int items = a.items * a.l.kv_heads;
    if ((int)blockIdx.x >= items) {  // the queries
        static_assert(sizeof xs >= kRopePairs * sizeof(float2));
        const int at = blockIdx.x - items, rows = (a.step.rows + a.rows_each - 1) / a.rows_each;
        const int row0 = at % rows * a.rows_each, head0 = at / rows * a.heads_each;
        const RopeRows g{a.q, a.q_out, a.q_stride, a.q_stride, D, a.bf16};
        const int n = min(a.rows_each, a.step.rows - row0), h = min(a.heads_each, a.heads - head0);
        if (a.wide) rope_rows<4>(g, a.rope, row0, n, head0, h, &a.step, (float2 *)xs);
        else rope_rows<1>(g, a.rope, row0, n, head0, h, &a.step, (float2 *)xs);
        return;
    }
    const int head = blockIdx.x % a.l.kv_heads;
    int blk = blockIdx.x / a.l.kv_heads, i;
    if (a.max_blocks) {
        i = blk / a.max_blocks;
        blk -= i * a.max_blocks;
    } else {
        i = sequence_of(a.step.block0, a.step.n, blk);
        blk -= a.step.block0[i];
    }
    const int row0 = a.step.row0[i], len = a.step.len[i], start = len - (a.step.row0[i + 1] - row0);
    const int b = start / kKvBlock + blk, lo = max(start, b * kKvBlock), hi = min(len, (b + 1) * kKvBlock);
    if (lo >= hi) return;
    const int page = a.step.table[(int64_t)a.step.seq[i] * a.step.sequence_pages + (b >> a.l.block_shift)];
    const int n = hi - lo, place = lo - b * kKvBlock;
    constexpr int X = (kKvBlock * D / 4 + 255) / 256, A = (kKvBlock * D / 2 + 255) / 256;  // pieces of a thread: values, angles
    float x[2][X][4];
    float2 cs[A];
    // t / pairs: half a step from a whole number is 2^-8 at least, and t is below 2^11
    const float per_pair = __builtin_amdgcn_rcpf((float)a.rope.pairs);
    auto row_of = [&](int t) { return (int)(((float)t + 0.5f) * per_pair); };
#pragma unroll
    for (int j = 0; j < X; j++) {
        const int t = tid + 256 * j, r = t / (D / 4), d = (t - r * (D / 4)) * 4;
        if (r >= n) break;
        const int64_t at = (int64_t)(row0 + lo - start + r) * a.kv_stride + head * D + d;
        load<4>(a.k, at, a.bf16 != 0, x[0][j]);
        load<4>(a.v, at, a.bf16 != 0, x[1][j]);
    }
    if (page < 0) return;
    const int in_page = (head << a.l.block_shift) + (b & ((1 << a.l.block_shift) - 1));
    uint8_t *pg = a.l.base + (int64_t)page * a.l.page_bytes;
    uint8_t *kc = pg + in_page * (2 * kKvBlock * D), *vc = kc + kKvBlock * D;
    float *sc = (float *)(pg + a.l.scales) + 2 * in_page;
    const float old_k = place ? sc[0] : 0.0f, old_v = place ? sc[1] : 0.0f;
    uint4 was_v = make_uint4(0, 0, 0, 0);
    if (tid < D && n < kKvBlock) was_v = *(const uint4 *)(vc + tid * kKvBlock);
    if (a.rope.pairs)
#pragma unroll
        for (int j = 0; j < A; j++) {
            const int t = tid + 256 * j, r = row_of(t);
            if (r >= n) break;
            cs[j] = turn_of(a.rope, t - r * a.rope.pairs, row0 + lo - start + r, lo + r);
        }
#pragma unroll
    for (int j = 0; j < X; j++) {
        const int t = tid + 256 * j, r = t / (D / 4), d = (t - r * (D / 4)) * 4;
        if (r >= n) break;
        *(float4 *)&xs[0][r][d] = make_float4(x[0][j][0], x[0][j][1], x[0][j][2], x[0][j][3]);
        *(float4 *)&xs[1][r][d] = make_float4(x[1][j][0], x[1][j][1], x[1][j][2], x[1][j][3]);
    }
    __syncthreads();
    if (a.rope.pairs) {
#pragma unroll
        for (int j = 0; j < A; j++) {
            const int t = tid + 256 * j, r = row_of(t), p = t - r * a.rope.pairs;
            if (r >= n) break;
            float *u = a.rope.interleaved ? &xs[0][r][2 * p] : &xs[0][r][p], *w = a.rope.interleaved ? u + 1 : u + a.rope.pairs;
            turn(cs[j].x, cs[j].y, *u, *w);
        }
        __syncthreads();
    }
    float mk = 0.0f, mv = 0.0f;
    for (int t = tid; t < n * D; t += 256) {
        const int r = t / D, d = t - r * D;
        const float k = fabsf(xs[0][r][d]), v = fabsf(xs[1][r][d]);
        mk = fmaxf(mk, k <= FLT_MAX ? k : __builtin_inff());
        mv = fmaxf(mv, v <= FLT_MAX ? v : __builtin_inff());
    }
    mk = block_max(mk, red[0]);
    mv = block_max(mv, red[1]);  // behind its barrier every thread has read the old scales
    float fk, fv;
    const float sk = next_scale(mk, place > 0, old_k, &fk), sv = next_scale(mv, place > 0, old_v, &fv);
    const float rk = sk == sk ? 1.0f / sk : 0.0f, rv = sv == sv ? 1.0f / sv : 0.0f;
    if (tid == 0) {
        sc[0] = sk;
        sc[1] = sv;
    }
    for (int t = tid; t < n * (D / 16); t += 256) {
        const int r = t / (D / 16), d = (t - r * (D / 16)) * 16;
        uint32_t w[4] = {0, 0, 0, 0};
        if (sk == sk)
            for (int j = 0; j < 16; j++) w[j / 4] |= code_of(xs[0][r][d + j], rk) << (j % 4 * 8);
        *(uint4 *)(kc + (place + r) * D + d) = make_uint4(w[0], w[1], w[2], w[3]);
    }
    if (fk < 1.0f)
        for (int t = tid; t < place * (D / 4); t += 256) {
            uint32_t *p = (uint32_t *)kc + t, o = 0;
            for (int j = 0; j < 4; j++) o |= shrink_of(*p >> (8 * j) & 0xff, fk) << (8 * j);
            *p = o;
        }
    if (const int d = tid; d < D) {
        uint4 *p = (uint4 *)(vc + d * kKvBlock);
        uint32_t w[4] = {was_v.x, was_v.y, was_v.z, was_v.w};
        for (int j = 0; j < kKvBlock; j++) {
            const int r = j - place;
            const uint32_t was = w[j / 4] >> (j % 4 * 8) & 0xff;
            uint32_t c = was;
            if (r < 0) c = fv < 1.0f ? shrink_of(was, fv) : was;
            else if (r < n) c = sv == sv ? code_of(xs[1][r][d], rv) : 0;
            w[j / 4] = (w[j / 4] & ~(0xffu << (j % 4 * 8))) | c << (j % 4 * 8);
        }
        *p = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// One block of 16 tokens of a kv head per workgroup.
template <int N>
__global__ void __launch_bounds__(256) read_kernel(KvReadOf<N> a, int blocks) {
    const int tid = threadIdx.x, D = a.l.dim, H = a.l.kv_heads;
    const int head = blockIdx.x % H, i = blockIdx.x / H / blocks;
    const int first = a.first[i], b = first / kKvBlock + blockIdx.x / H % blocks;
    const int64_t end = first + a.count;
    const int lo = max(first, b * kKvBlock), hi = (int)min(end, (int64_t)(b + 1) * kKvBlock);
    if (lo >= hi) return;
    __shared__ uint8_t vt[kKvMaxDim][kKvBlock + 4];
    const int page = b * kKvBlock < a.len[i] ? a.table[(int64_t)a.seq[i] * a.sequence_pages + (b >> a.l.block_shift)] : -1;
    const int in_page = (head << a.l.block_shift) + (b & ((1 << a.l.block_shift) - 1));
    const uint8_t *pg = a.l.base + (int64_t)max(page, 0) * a.l.page_bytes, *kc = pg + in_page * (2 * kKvBlock * D), *vc = kc + kKvBlock * D;
    float sk = 0.0f, sv = 0.0f;
    if (page >= 0) {
        const float *sc = (const float *)(pg + a.l.scales) + 2 * in_page;
        sk = sc[0], sv = sc[1];
        for (int d = tid; d < D; d += 256) {
            const uint4 v = *(const uint4 *)(vc + d * kKvBlock);
            uint32_t *o = (uint32_t *)vt[d];
            o[0] = v.x, o[1] = v.y, o[2] = v.z, o[3] = v.w;
        }
    }
    __syncthreads();
    for (int t = tid; t < (hi - lo) * (D / 4); t += 256) {
        const int r = t / (D / 4), d = (t - r * (D / 4)) * 4, p = lo + r, j = p - b * kKvBlock;
        float4 k = make_float4(0, 0, 0, 0), v = k;
        if (page >= 0 && p < a.len[i]) {
            const char4 c = *(const char4 *)(kc + j * D + d);
            k = make_float4(c.x * sk, c.y * sk, c.z * sk, c.w * sk);
            v = make_float4((int8_t)vt[d][j] * sv, (int8_t)vt[d + 1][j] * sv, (int8_t)vt[d + 2][j] * sv, (int8_t)vt[d + 3][j] * sv);
        }
        const int64_t at = (((int64_t)i * a.count + (p - first)) * H + head) * D + d;
        if (a.k) *(float4 *)(a.k + at) = k;
        if (a.v) *(float4 *)(a.v + at) = v;
    }
}

// A wave per run.
template <int N>
__global__ void __launch_bounds__(64) runs_kernel(KvRunsOf<N> a) {
    const KvRun r = a.run[blockIdx.x];
    for (int j = threadIdx.x; j < r.count; j += 64) a.words[r.at + j] = r.value + r.step * j;
}

// 16 KiB of a page per workgroup, four loads of a thread on their way before the first store.
constexpr int kCopyBytes = 16384;
template <int N>
__global__ void __launch_bounds__(256) copy_kernel(KvPairsOf<N> a) {
    uint8_t *base = a.pool + (int64_t)blockIdx.z * a.layer_bytes;
    const uint4 *src = (const uint4 *)(base + (int64_t)a.src[blockIdx.y] * a.page_bytes);
    uint4 *dst = (uint4 *)(base + (int64_t)a.dst[blockIdx.y] * a.page_bytes);
    const int last = (int)(a.page_bytes / 16) - 1, at = blockIdx.x * (kCopyBytes / 16) + threadIdx.x;
    // behind the page's end its last piece again
    const int i0 = min(at, last), i1 = min(at + 256, last), i2 = min(at + 512, last), i3 = min(at + 768, last);
    const uint4 v0 = src[i0], v1 = src[i1], v2 = src[i2], v3 = src[i3];
    dst[i0] = v0;
    dst[i1] = v1;
    dst[i2] = v2;
    dst[i3] = v3;
}

}  // namespace

hipError_t launch_rope(const void *x, void *out, int64_t rows, int32_t heads, int32_t dim, int64_t stride, int64_t out_stride, bool bf16,
                       const KvRope &rope, hipStream_t s) {
    const uintptr_t e = bf16 ? 2 : 4;
    const auto wide = [&](int v) {  // v values a load, of at most 16 bytes
        const uintptr_t bytes = v * e;
        return dim % (2 * v) == 0 && rope.pairs % v == 0 && (uintptr_t)x % bytes == 0 && (uintptr_t)out % bytes == 0 && stride * e % bytes == 0 &&
               out_stride * e % bytes == 0;
    };
    const int v = bf16 && wide(8) ? 8 : wide(4) ? 4 : 1;
    const RopeGrid g = rope_grid(rows, heads, dim, v, rope.pairs);
    if (g.groups_x > INT32_MAX || g.groups_y > 65535) return hipErrorInvalidValue;
    const RopeRows r{x, out, stride, out_stride, dim, bf16};
    const dim3 grid((unsigned)g.groups_x, (unsigned)g.groups_y);
    if (v == 8) rope_kernel<8><<<grid, 256, 0, s>>>(r, rows, heads, g.rows, g.heads, rope);
    else if (v == 4) rope_kernel<4><<<grid, 256, 0, s>>>(r, rows, heads, g.rows, g.heads, rope);
    else rope_kernel<1><<<grid, 256, 0, s>>>(r, rows, heads, g.rows, g.heads, rope);
    return hipGetLastError();
}

hipError_t launch_kv_append(const KvAppend &args, hipStream_t s, hipEvent_t done) {
    KvAppend a = args;
    const int64_t items = (int64_t)a.items * a.l.kv_heads;
    int64_t q = 0;
    if (a.heads) {
        a.wide = a.rope.pairs % 4 == 0;
        const RopeGrid g = rope_grid(a.step.rows, a.heads, a.l.dim, a.wide ? 4 : 1, a.rope.pairs);
        a.rows_each = g.rows;
        a.heads_each = g.heads;
        q = g.groups_x * g.groups_y;
    }
    if (items + q > INT32_MAX) return hipErrorInvalidValue;
    const dim3 grid((unsigned)(items + q));
    switch (a.l.dim) {
    case 64: return launch_with_event(append_kernel<64>, grid, dim3(256), s, done, a);
    case 96: return launch_with_event(append_kernel<96>, grid, dim3(256), s, done, a);
    case 128: return launch_with_event(append_kernel<128>, grid, dim3(256), s, done, a);
    case 192: return launch_with_event(append_kernel<192>, grid, dim3(256), s, done, a);
    case 256: return launch_with_event(append_kernel<256>, grid, dim3(256), s, done, a);
    }
    return hipErrorInvalidValue;
}

hipError_t launch_kv_read(const KvRead &r, hipStream_t s, hipEvent_t done) {
    const int blocks = (int)((r.count + 2 * kKvBlock - 2) / kKvBlock);
    const dim3 grid((unsigned)(r.n * blocks * r.l.kv_heads));
    if (r.n > 64) return launch_with_event(read_kernel<kKvReadSeqs>, grid, dim3(256), s, done, r, blocks);
    KvReadOf<64> few{r.l, r.table, r.sequence_pages, r.n, r.count, r.k, r.v};
    std::copy_n(r.seq, r.n, few.seq);
    std::copy_n(r.first, r.n, few.first);
    std::copy_n(r.len, r.n, few.len);
    return launch_with_event(read_kernel<64>, grid, dim3(256), s, done, few, blocks);
}

hipError_t launch_kv_runs(const KvRuns &r, hipStream_t s, hipEvent_t done) {
    const dim3 grid((unsigned)r.n);
    if (r.n > 24) return launch_with_event(runs_kernel<kKvRuns>, grid, dim3(64), s, done, r);
    KvRunsOf<24> few{r.words, r.n};
    std::copy_n(r.run, r.n, few.run);
    return launch_with_event(runs_kernel<24>, grid, dim3(64), s, done, few);
}

hipError_t launch_kv_copy(const KvPairs &p, hipStream_t s, hipEvent_t done) {
    const dim3 grid((unsigned)((p.page_bytes + kCopyBytes - 1) / kCopyBytes), (unsigned)p.n, (unsigned)p.layers);
    if (p.n > 48) return launch_with_event(copy_kernel<kKvPairs>, grid, dim3(256), s, done, p);
    KvPairsOf<48> few{p.pool, p.page_bytes, p.layer_bytes, p.layers, p.n};
    std::copy_n(p.src, p.n, few.src);
    std::copy_n(p.dst, p.n, few.dst);
    return launch_with_event(copy_kernel<48>, grid, dim3(256), s, done, few);
}

}  // namespace j4q
