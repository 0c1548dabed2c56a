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
// A value that is not finite makes the whole block of its head NaN: the cache has no code for it, and NaN is not lost.
#include "kv.h"

#include <float.h>

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

// Cosines and sines of pairs [pair, pair + V) of row `row`, which is token `place` of its sequence.
template <int V>
__device__ __forceinline__ void turns_of(const KvRope &r, int pair, int64_t row, int place, float *c, float *s) {
    int at[V];
    if (r.axes > 1) {
#pragma unroll
        for (int j = 0; j < V; j++) at[j] = r.positions[(int64_t)r.axis[pair + j] * r.rows + row];
    } else {
        const int one = r.positions ? r.positions[row] : place;
#pragma unroll
        for (int j = 0; j < V; j++) at[j] = one;
    }
#pragma unroll
    for (int j = 0; j < V; j++) {
        const bool there = at[j] >= 0 && at[j] < r.table_rows;  // else no angle in the tables
        const int64_t i = (int64_t)(there ? at[j] : 0) * r.pairs + pair + j;
        c[j] = there ? r.cos[i] : __builtin_nanf("");
        s[j] = there ? r.sin[i] : __builtin_nanf("");
    }
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

// 2 V channels of H heads of a row from head0 on: V pairs that are turned, by the same cosines and sines for every head, or channels behind
// those, which are copied. unit: which of the dim / (2 V). All loads go out before the first is used. In place is fine: a
// thread reads what it writes.
template <int V, int H>
__device__ __forceinline__ void rope_unit(const void *x, void *out, int64_t in_row, int64_t out_row, int head0, int dim, int unit, bool bf16,
                                          const KvRope &r, int64_t row, int place) {
    const int i = unit * V;
    const bool turned = i < r.pairs;
    const int at0 = turned && !r.interleaved ? i : 2 * i, at1 = turned && !r.interleaved ? i + r.pairs : 2 * i + V;
    float a[H][2][V], c[V], s[V];
#pragma unroll
    for (int h = 0; h < H; h++) {
        const int64_t from = in_row + (int64_t)(head0 + h) * dim;
        load<V>(x, from + at0, bf16, a[h][0]);
        load<V>(x, from + at1, bf16, a[h][1]);
    }
    if (turned) turns_of<V>(r, i, row, place, c, s);
#pragma unroll
    for (int h = 0; h < H; h++) {
        if (turned) {
            float *f = &a[h][0][0];
            if (r.interleaved) {
#pragma unroll
                for (int j = 0; j < V; j++) turn(c[j], s[j], f[2 * j], f[2 * j + 1]);
            } else {
#pragma unroll
                for (int j = 0; j < V; j++) turn(c[j], s[j], f[j], f[V + j]);
            }
        }
        const int64_t to = out_row + (int64_t)(head0 + h) * dim;
        store<V>(out, to + at0, bf16, a[h][0]);
        store<V>(out, to + at1, bf16, a[h][1]);
    }
}

template <int V, int H>
__global__ void __launch_bounds__(256)
rope_kernel(const void *x, void *out, int64_t rows, int heads, int dim, int64_t stride, int64_t out_stride, int bf16, KvRope r) {
    const int units = dim / (2 * V), parts = heads / H;
    const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t row = t / (units * parts);
    if (row >= rows) return;
    const int rest = (int)(t - row * (units * parts)), part = rest / units;
    rope_unit<V, H>(x, out, row * stride, row * out_stride, part * H, dim, rest - part * units, bf16 != 0, r, row, (int)row);
}

__device__ __forceinline__ float block_max(float v, float *red) {
    for (int d = 32; d; d >>= 1) v = fmaxf(v, __shfl_xor(v, d));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
}

// The block's scale after values of magnitude up to amax, and 2^-k for the codes that are there.
__device__ __forceinline__ float next_scale(float amax, bool begun, float old, float *shrink) {
    *shrink = 1.0f;
    if (!(amax <= FLT_MAX)) return __builtin_nanf("");
    if (begun && old != old) return old;
    if (!begun || old <= kKvMinScale) return fmaxf(amax / 127.0f, kKvMinScale);
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

// One block of 16 tokens of a kv head per workgroup, 256 threads; the workgroups behind them turn the queries.
template <int D>
__global__ void __launch_bounds__(256) append_kernel(KvAppend a) {
    constexpr int P = D + 4;
    __shared__ float xs[2][kKvBlock][P];
    __shared__ float red[2][4];
    const int tid = threadIdx.x;
    const int items = a.items * a.l.kv_heads;
    if ((int)blockIdx.x >= items) {  // 4 pairs of one or four query heads a thread
        const int units = D / 8, parts = a.heads / a.heads_each;
        const int64_t t = (int64_t)(blockIdx.x - items) * 256 + tid, row = t / (units * parts);
        if (row >= a.step.rows) return;
        const int rest = (int)(t - row * (units * parts)), head = rest / units * a.heads_each, unit = rest % units;
        int place = 0;
        if (a.rope.pairs && !a.rope.positions) {
            const int i = sequence_of(a.step.row0, a.step.n, (int)row);
            place = a.step.len[i] - a.step.row0[i + 1] + (int)row;
        }
        const int64_t at = row * a.q_stride;
        if (a.rope.pairs % 4 != 0) {
            for (int j = 0; j < 4; j++)
                for (int h = 0; h < a.heads_each; h++) rope_unit<1, 1>(a.q, a.q_out, at, at, head + h, D, unit * 4 + j, a.bf16 != 0, a.rope, row, place);
        } else if (a.heads_each == 4) {
            rope_unit<4, 4>(a.q, a.q_out, at, at, head, D, unit, a.bf16 != 0, a.rope, row, place);
        } else {
            rope_unit<4, 1>(a.q, a.q_out, at, at, head, D, unit, a.bf16 != 0, a.rope, row, place);
        }
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
    if (page < 0) return;
    const int n = hi - lo, place = lo - b * kKvBlock;
    const int in_page = (head << a.l.block_shift) + (b & ((1 << a.l.block_shift) - 1));
    uint8_t *pg = a.l.base + (int64_t)page * a.l.page_bytes;
    uint8_t *kc = pg + in_page * (2 * kKvBlock * D), *vc = kc + kKvBlock * D;
    float *sc = (float *)(pg + a.l.scales) + 2 * in_page;
    const float old_k = place ? sc[0] : 0.0f, old_v = place ? sc[1] : 0.0f;
    for (int t = tid; t < n * (D / 4); t += 256) {
        const int r = t / (D / 4), d = (t - r * (D / 4)) * 4;
        const int64_t at = (int64_t)(row0 + lo - start + r) * a.kv_stride + head * D + d;
        load<4>(a.k, at, a.bf16 != 0, &xs[0][r][d]);
        load<4>(a.v, at, a.bf16 != 0, &xs[1][r][d]);
    }
    __syncthreads();
    if (a.rope.pairs) {
        for (int t = tid; t < n * a.rope.pairs; t += 256) {
            const int r = t / a.rope.pairs, p = t - r * a.rope.pairs;
            float c, s;
            turns_of<1>(a.rope, p, row0 + lo - start + r, lo + r, &c, &s);
            float *u = a.rope.interleaved ? &xs[0][r][2 * p] : &xs[0][r][p], *w = a.rope.interleaved ? u + 1 : u + a.rope.pairs;
            turn(c, s, *u, *w);
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
    for (int d = tid; d < D; d += 256) {
        uint4 *p = (uint4 *)(vc + d * kKvBlock);
        uint4 o = make_uint4(0, 0, 0, 0);
        if (n < kKvBlock) o = *p;
        uint32_t w[4] = {o.x, o.y, o.z, o.w};
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
__global__ void __launch_bounds__(256) read_kernel(KvRead a, int blocks) {
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
__global__ void __launch_bounds__(64) runs_kernel(KvRuns a) {
    const KvRun r = a.run[blockIdx.x];
    for (int j = threadIdx.x; j < r.count; j += 64) a.words[r.at + j] = r.value + r.step * j;
}

// 16 KiB of a page per workgroup, four loads of a thread on their way before the first store.
constexpr int kCopyBytes = 16384;
__global__ void __launch_bounds__(256) copy_kernel(KvPairs a) {
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
        const uintptr_t bytes = v * e < 16 ? v * e : 16;
        return dim % (2 * v) == 0 && rope.pairs % v == 0 && (uintptr_t)x % bytes == 0 && (uintptr_t)out % bytes == 0 && stride * e % bytes == 0 &&
               out_stride * e % bytes == 0;
    };
    const int v = bf16 && wide(8) ? 8 : wide(4) ? 4 : 1;
    // four heads a thread share its cosines and sines, where that leaves threads for the chip
    const int h = v > 1 && heads % 4 == 0 && rows * heads * (dim / (2 * v)) >= 1 << 18 ? 4 : 1;
    const dim3 grid((unsigned)((rows * (heads / h) * (dim / (2 * v)) + 255) / 256));
    const auto run = [&](auto kernel) { kernel<<<grid, 256, 0, s>>>(x, out, rows, heads, dim, stride, out_stride, bf16, rope); };
    if (v == 8) h == 4 ? run(rope_kernel<8, 4>) : run(rope_kernel<8, 1>);
    else if (v == 4) h == 4 ? run(rope_kernel<4, 4>) : run(rope_kernel<4, 1>);
    else run(rope_kernel<1, 1>);
    return hipGetLastError();
}

hipError_t launch_kv_append(const KvAppend &args, hipStream_t s, hipEvent_t done) {
    KvAppend a = args;
    const int64_t items = (int64_t)a.items * a.l.kv_heads;
    a.heads_each = a.heads % 4 == 0 && (int64_t)a.step.rows * a.heads * (a.l.dim / 8) >= 1 << 18 ? 4 : 1;
    const int64_t q = ((int64_t)a.step.rows * (a.heads / a.heads_each) * (a.l.dim / 8) + 255) / 256;
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
    return launch_with_event(read_kernel, dim3((unsigned)(r.n * blocks * r.l.kv_heads)), dim3(256), s, done, r, blocks);
}

hipError_t launch_kv_runs(const KvRuns &r, hipStream_t s, hipEvent_t done) {
    return launch_with_event(runs_kernel, dim3((unsigned)r.n), dim3(64), s, done, r);
}

hipError_t launch_kv_copy(const KvPairs &p, hipStream_t s, hipEvent_t done) {
    const dim3 grid((unsigned)((p.page_bytes + kCopyBytes - 1) / kCopyBytes), (unsigned)p.n, (unsigned)p.layers);
    return launch_with_event(copy_kernel, grid, dim3(256), s, done, p);
}

}  // namespace j4q
