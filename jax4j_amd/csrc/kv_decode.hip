// Attention over the 8-bit cache where a sequence has few query rows (decoding): up to 8 rows (tokens x query heads of a kv
// head) per workgroup, so memory bounds it: 2 D + 1/2 bytes of a token and kv head are read once.
//
// For a row with query q, a token j with codes k_j, v_j of blocks with scales sk, sv:
//   t_j = scale * log2(e) * sk (q . k_j) + log2(sv)       w_j = 2^(t_j - m + 26)       m >= every t_j so far - 4
//   out = sum_j w_j v_j / sum_j w_j / sv
// The value scale goes into the exponent, so that w times the plain codes is the weighted sum; the sum of the weights alone
// divides it out again. A visible token of a block of NaN has t = NaN, and so has its row.
//
// Both products run on the int8 matrix instruction 16x16x64 over the codes as they lie in memory, with exact 32-bit sums.
// The other operand is fp32 (q, w); it enters as four digits to the base 256 from -128 to 127 of a whole number of 31 bits: q over
// its row's largest magnitude / 2^30, so nothing that fp32 holds beside that is lost; w below 2^30, rounded to the nearest, so a
// weight is off by 2^-27 of the largest that its wave has seen at most, either way (cut off, thousands of tokens far below a
// dominant one lost half a unit each: 0.6 to 1.2 % of their sum). The digits fill the 16 columns of the second operand: 4 rows x
// 4 digits in one instruction, or 8 rows x 2 digits in two. Operands:
//   scores   A = 16 tokens x 64 channels of K, B = 64 channels x 16 (digit, row):  C[token][digit, row]
//   output   A = 16 channels x 64 tokens of V, B = 64 tokens x 16 (digit, row) of w: C[channel][digit, row]
// Lane l holds rows 4 (l / 16) + i of C in column l % 16, bytes 16 (l / 16).. of k in A's row and B's column l % 16. The 16
// tokens of score product s = 0..3 are numbered 16 (m / 4) + 4 s + m % 4 by their row m, so that a lane's 16 scores are those of
// block l / 16 of the tile, in order: they become its bytes of B, under one pair of scales, without leaving the lane.
//
// The 32-bit sums of an output stay in the matrix instruction's accumulators over tiles for as long as no t passes m + 4 (m then
// moves up, the sums go to fp32 and start again), so a tile costs no vector instruction per output. 2^26 x 127 x digits: 65536
// tokens stay below 2^31 in every digit.
//
// A wave walks tiles of its own, loaded a tile ahead into registers, so that nothing but the last sum goes through LDS and no wave
// waits for another. 8 kv heads of 128, 32 query heads, fp32: 64 sequences of up to 8191 tokens (681 MB) 115 us, 5.9 TB/s, where
// a plain read reaches 6.0; 131071 tokens of one (269 MB), 32 ranges, 51 us and 5 to join them; 293 tokens 8, the latency of
// one tile. 32 sequences in a window of 1024, heads of 64 (34 MB): 10 us.
#include "kv.h"

namespace j4q {
namespace {

typedef int v4i __attribute__((ext_vector_type(4)));

constexpr float kHead = 4.0f;    // octaves that t may pass m by
constexpr float kUnit = 26.0f;   // 2^26: the weight of t = m
constexpr int kFlushTiles = 1024;

// v + the lanes' that are N to the right in their 16, round about.
template <int N>
__device__ __forceinline__ float add_ror(float v) {
    return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x120 + N, 0xf, 0xf, true));
}
// Over the columns that hold digits of the same row.
template <int R>
__device__ __forceinline__ float sum_digits(float v) {
    v = add_ror<8>(v);
    if constexpr (R == 4) v = add_ror<4>(v);
    return v;
}
// Over the four lanes of a column. A swap gives every lane its own value and the one across, in two registers; the compiler
// takes them for the same where both operands are, so one of them is a copy that it cannot see through.
struct Two {
    float a, b;
};
__device__ __forceinline__ Two swap32(float v) {
    uint32_t x = __builtin_bit_cast(uint32_t, v), y = x;
    asm("" : "+v"(y));
    const auto r = __builtin_amdgcn_permlane32_swap(x, y, false, false);
    return {__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1])};
}
__device__ __forceinline__ Two swap16(float v) {
    uint32_t x = __builtin_bit_cast(uint32_t, v), y = x;
    asm("" : "+v"(y));
    const auto r = __builtin_amdgcn_permlane16_swap(x, y, false, false);
    return {__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1])};
}
__device__ __forceinline__ float max_column(float v) {
    const Two a = swap32(v);
    const Two b = swap16(fmaxf(a.a, a.b));
    return fmaxf(b.a, b.b);
}
__device__ __forceinline__ float sum_column(float v) {
    const Two a = swap32(v);
    const Two b = swap16(a.a + a.b);
    return b.a + b.b;
}

__device__ __forceinline__ uint32_t digits_of(int v) { return (uint32_t)v + 0x80808080u; }  // each byte its digit + 128
// Byte `digit` of four of them, as signed bytes.
__device__ __forceinline__ int pick(uint32_t a, uint32_t b, uint32_t c, uint32_t d, uint32_t low, uint32_t high) {
    return (int)((__builtin_amdgcn_perm(b, a, low) | __builtin_amdgcn_perm(d, c, high)) ^ 0x80808080u);
}

// 16 values from i on, 16-byte aligned.
__device__ __forceinline__ void load16(const void *p, int64_t i, int bf16, float *x) {
    if (bf16) {
        const uint4 *from = (const uint4 *)((const uint16_t *)p + i);
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const uint4 t = from[j];
            const uint32_t w[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
            for (int e = 0; e < 4; e++) {
                x[8 * j + 2 * e] = __builtin_bit_cast(float, w[e] << 16);
                x[8 * j + 2 * e + 1] = __builtin_bit_cast(float, w[e] & 0xffff0000u);
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float4 t = ((const float4 *)((const float *)p + i))[j];
            x[4 * j] = t.x, x[4 * j + 1] = t.y, x[4 * j + 2] = t.z, x[4 * j + 3] = t.w;
        }
    }
}
__device__ __forceinline__ void store_out(void *p, int64_t i, int bf16, float f) {
    if (bf16) {
        const uint32_t u = __builtin_bit_cast(uint32_t, f);
        ((uint16_t *)p)[i] = f != f ? (uint16_t)((u >> 16) | 0x40) : (uint16_t)((u + 0x7fffu + ((u >> 16) & 1)) >> 16);
    } else {
        ((float *)p)[i] = f;
    }
}

// Waves of a workgroup, each with its own tiles: two on a SIMD where their registers allow.
constexpr int waves_of(int d) { return d > 128 ? 4 : 8; }

template <int D, int R>
__global__ void __launch_bounds__(64 * waves_of(D), waves_of(D) / 4) decode_kernel(KvAttend a) {
    constexpr int kWaves = waves_of(D);
    constexpr int M = R / 4;                // matrix instructions for the four digits
    constexpr int S = (D + 63) / 64;        // steps of 64 channels
    constexpr int T = D / 16;               // tiles of 16 channels of the output
    __shared__ float part[kWaves][R][D];
    __shared__ float part_ml[kWaves][R][2];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, quad = lane >> 4;
    const int i = blockIdx.z, head = blockIdx.y % a.l.kv_heads, rg = blockIdx.y / a.l.kv_heads;
    const int row0 = a.step.row0[i], tokens = a.step.row0[i + 1] - row0, len = a.step.len[i];
    if (rg * R >= tokens * a.group || tokens * a.group > a.rows_to) return;
    // tokens of this workgroup's rows
    const int q_first = len - tokens + rg * R / a.group, q_last = len - tokens + min(tokens * a.group - 1, rg * R + R - 1) / a.group;
    const KvTiles vis = kv_tiles(q_first, q_last, a.window, a.sinks);
    int t0 = 0, t1 = vis.count();
    if (a.splits > 1) {
        const int each = kv_range_tiles(t1, a);
        t0 = blockIdx.x * each;
        if (t0 >= t1) return;
        t1 = min(t1, t0 + each);
    }

    const int32_t *table = a.step.table + (int64_t)a.step.seq[i] * a.step.sequence_pages;
    const int last_block = (len - 1) / kKvBlock, in_page = (1 << a.l.block_shift) - 1;
    const uint32_t block_bytes = 2 * kKvBlock * D;

    v4i kr[4][S], vr[T];
    float2 sc;
    // Pages of the lane's block of K and of V in a tile, looked up a tile ahead of the loads from them. A page that is not there
    // gives bytes that weigh nothing.
    int page_k, page_v;
    auto look_up = [&](int tile) {
        page_k = table[min(tile * 4 + (col >> 2), last_block) >> a.l.block_shift];
        page_v = table[min(tile * 4 + quad, last_block) >> a.l.block_shift];
    };
    auto block_at = [&](int tile, int b, int page, int *in) -> const uint8_t * {
        *in = (head << a.l.block_shift) + (min(tile * 4 + b, last_block) & in_page);
        return a.l.base + (int64_t)max(page, 0) * a.l.page_bytes;
    };
    auto load_k = [&](int tile) {
        int in;
        const uint8_t *pg = block_at(tile, col >> 2, page_k, &in), *k = pg + in * block_bytes + (col & 3) * D + quad * 16;
#pragma unroll
        for (int s = 0; s < 4; s++)
#pragma unroll
            for (int c = 0; c < S; c++) kr[s][c] = *(const v4i *)(k + 4 * s * D + 64 * c);
    };
    auto load_v = [&](int tile) {
        int in;
        const uint8_t *pg = block_at(tile, quad, page_v, &in), *v = pg + in * block_bytes + kKvBlock * D + col * 16;
        sc = *(const float2 *)(pg + a.l.scales + 8 * in);
#pragma unroll
        for (int t = 0; t < T; t++) vr[t] = *(const v4i *)(v + 256 * t);
    };

    // the wave's first tile, while the queries are made ready
    if (t0 + wave < t1) {
        const int tile = vis.tile(t0 + wave);
        look_up(tile);
        load_k(tile);
        load_v(tile);
        if (t0 + wave + kWaves < t1) look_up(vis.tile(t0 + wave + kWaves));
    }

    const int rr = min(rg * R + col % R, tokens * a.group - 1);  // a column that is no row's has the last row's
    const int p = len - tokens + rr / a.group;               // the row's place
    const int first_low = max(p - a.window + 1, 0);          // its first token behind the window's edge
    // the row's digits: column col holds digit col / R (+ 2 in a second instruction)
    int qd[M][S][4];
    float weight[M];
    float q_scale;
    {
        const int64_t at = (int64_t)(row0 + rr / a.group) * a.q_stride + (head * a.group + rr % a.group) * D;
        float x[S][16], most = 0.0f, finite = 0.0f;
#pragma unroll
        for (int s = 0; s < S; s++) {
            const int d = s * 64 + quad * 16;
            if (d < D) {
                load16(a.q, at + d, a.q_bf16, x[s]);
            } else {
                for (int j = 0; j < 16; j++) x[s][j] = 0.0f;
            }
#pragma unroll
            for (int j = 0; j < 16; j++) {
                most = fmaxf(most, fabsf(x[s][j]));
                finite = __builtin_fmaf(x[s][j], 0.0f, finite);  // else NaN
            }
        }
        most = max_column(most);
        finite = sum_column(finite);
        // at least 2^-90, so that its reciprocal is finite
        const float unit = fmaxf(most, 0x1p-90f) * 0x1p-30f, inv = 1.0f / unit;
        q_scale = unit * a.scale + finite;
        for (int m = 0; m < M; m++) {
            const uint32_t digit = (16 / R) * m + col / R;
            const uint32_t low = digit | (digit + 4) << 8 | 0x0c0c0000u, high = 0x0c0cu | digit << 16 | (digit + 4) << 24;
            weight[m] = __builtin_bit_cast(float, (127 + 8 * digit) << 23);
            for (int s = 0; s < S; s++)
                for (int j = 0; j < 4; j++)
                    qd[m][s][j] = pick(digits_of((int)(x[s][4 * j] * inv)), digits_of((int)(x[s][4 * j + 1] * inv)),
                                       digits_of((int)(x[s][4 * j + 2] * inv)), digits_of((int)(x[s][4 * j + 3] * inv)), low, high);
        }
    }

    v4i acc[M][T];
    float o[T][4], m_at = -__builtin_inff(), l_sum = 0.0f;
    for (int t = 0; t < T; t++) {
        for (int m = 0; m < M; m++) acc[m][t] = v4i{0, 0, 0, 0};
        for (int j = 0; j < 4; j++) o[t][j] = 0.0f;
    }
    int since = 0;
    for (int u = t0 + wave; u < t1; u += kWaves) {
        const int tile = vis.tile(u);
        const bool more = u + kWaves < t1;
        float t[16];
        float sk = sc.x, sv = fmaxf(sc.y, kKvMinScale);
        if (sc.y != sc.y) sv = sc.y;
        if (tile * 4 + quad > last_block) sk = 0.0f, sv = 1.0f;  // behind the end
        const float lv = __builtin_amdgcn_logf(sv), rsv = sv == sv ? 1.0f / sv : 1.0f;
        const float qk = q_scale * sk;
        float top = -__builtin_inff();
#pragma unroll
        for (int s = 0; s < 4; s++) {
            v4i c[M];
#pragma unroll
            for (int m = 0; m < M; m++) {
                c[m] = v4i{0, 0, 0, 0};
#pragma unroll
                for (int st = 0; st < S; st++)
                    c[m] = __builtin_amdgcn_mfma_i32_16x16x64_i8(kr[s][st], v4i{qd[m][st][0], qd[m][st][1], qd[m][st][2], qd[m][st][3]}, c[m], 0, 0, 0);
            }
#pragma unroll
            for (int j = 0; j < 4; j++) {
                float x = (float)c[0][j] * weight[0];
                if constexpr (M > 1) x = __builtin_fmaf((float)c[1][j], weight[1], x);
                t[4 * s + j] = __builtin_fmaf(sum_digits<R>(x), qk, lv);
            }
        }
        if (more) load_k(vis.tile(u + kWaves));
        // tokens that not every row sees
        const int j0 = tile * kKvTile;
        if (j0 + kKvTile - 1 > q_first || (j0 <= q_last - a.window && j0 + kKvTile - 1 >= a.sinks)) {
            const int at = j0 + quad * kKvBlock;
#pragma unroll
            for (int j = 0; j < 16; j++) {
                const bool seen = (at + j <= p) & ((at + j >= first_low) | (at + j < a.sinks));
                t[j] = seen ? t[j] : -__builtin_inff();
            }
        }
#pragma unroll
        for (int j = 0; j < 16; j++) top = fmaxf(top, t[j]);
        top = max_column(top);
        // by all four digits' columns alike: their t are the same bits
        if (__any(top > m_at + kHead) || ++since == kFlushTiles) {
            since = 0;
            const float to = fmaxf(top > m_at + kHead ? top : m_at, m_at), f = to > m_at ? __builtin_amdgcn_exp2f(m_at - to) : 1.0f;
            m_at = to;
            l_sum *= f;
            if (u >= t0 + kWaves) {  // before, there is nothing to scale
#pragma unroll
                for (int tt = 0; tt < T; tt++)
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        float x = (float)acc[0][tt][j] * weight[0];
                        if constexpr (M > 1) x = __builtin_fmaf((float)acc[1][tt][j], weight[1], x);
                        o[tt][j] = (o[tt][j] + x) * f;
#pragma unroll
                        for (int m = 0; m < M; m++) acc[m][tt][j] = 0;
                    }
            }
        }
        const float base = m_at > -__builtin_inff() ? kUnit - m_at : 0.0f;
        uint32_t w[16];
#pragma unroll
        for (int j = 0; j < 16; j++) {
            const float e = __builtin_amdgcn_exp2f(t[j] + base);
            l_sum = __builtin_fmaf(e, rsv, l_sum);
            w[j] = digits_of((int)__builtin_rintf(e));
        }
#pragma unroll
        for (int m = 0; m < M; m++) {
            const uint32_t digit = (16 / R) * m + col / R;
            const uint32_t low = digit | (digit + 4) << 8 | 0x0c0c0000u, high = 0x0c0cu | digit << 16 | (digit + 4) << 24;
            v4i b;
#pragma unroll
            for (int s = 0; s < 4; s++) b[s] = pick(w[4 * s], w[4 * s + 1], w[4 * s + 2], w[4 * s + 3], low, high);
#pragma unroll
            for (int tt = 0; tt < T; tt++) acc[m][tt] = __builtin_amdgcn_mfma_i32_16x16x64_i8(vr[tt], b, acc[m][tt], 0, 0, 0);
        }
        if (more) {
            load_v(vis.tile(u + kWaves));
            if (u + 2 * kWaves < t1) look_up(vis.tile(u + 2 * kWaves));
        }
    }

    l_sum = sum_column(l_sum);
#pragma unroll
    for (int t = 0; t < T; t++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            float x = (float)acc[0][t][j] * weight[0];
            if constexpr (M > 1) x = __builtin_fmaf((float)acc[1][t][j], weight[1], x);
            x = sum_digits<R>(o[t][j] + x);
            if (col < R) part[wave][col][16 * t + 4 * quad + j] = x;
        }
    if (lane < R) {
        part_ml[wave][lane][0] = m_at;
        part_ml[wave][lane][1] = l_sum;
    }
    __syncthreads();
    for (int at = threadIdx.x; at < R * D; at += 64 * kWaves) {
        const int r = at / D, d = at - r * D, row = rg * R + r;
        if (row >= tokens * a.group) break;
        float most = part_ml[0][r][0];
        for (int w = 1; w < kWaves; w++) most = fmaxf(most, part_ml[w][r][0]);
        float sum = 0.0f, total = 0.0f;
        if (most > -__builtin_inff())
            for (int w = 0; w < kWaves; w++) {
                const float f = __builtin_amdgcn_exp2f(part_ml[w][r][0] - most);
                sum = __builtin_fmaf(part[w][r][d], f, sum);
                total = __builtin_fmaf(part_ml[w][r][1], f, total);
            }
        else
            for (int w = 0; w < kWaves; w++) total += part_ml[w][r][1];  // NaN where every t was
        if (a.splits > 1) {
            const int64_t slot = (((int64_t)i * a.l.kv_heads + head) * a.max_rows + row) * a.splits + blockIdx.x;
            a.part[slot * D + d] = sum;
            if (d == 0) {
                a.part_ml[2 * slot] = most;
                a.part_ml[2 * slot + 1] = total;
            }
        } else {
            const int64_t to = (int64_t)(row0 + row / a.group) * a.out_stride + (head * a.group + row % a.group) * D + d;
            store_out(a.out, to, a.out_bf16, total == 0.0f ? 0.0f : sum / total);
        }
    }
}

// A row per workgroup: D / 4 threads for four channels each, as many of these as 256 threads hold for ranges of their own, whose
// first parts are on their way while the largest max is found. (One thread per channel that walked all ranges: 23 us for 64
// ranges, a load's latency each.)
__global__ void __launch_bounds__(256) join_kernel(KvAttend a) {
    constexpr int kAhead = 8, kRanges = kKvSplits;
    __shared__ float fs[kRanges], red[2][4];
    __shared__ float4 sums[256];
    const int i = blockIdx.z, head = blockIdx.y, row = blockIdx.x, D = a.l.dim, tid = threadIdx.x;
    const int row0 = a.step.row0[i], tokens = a.step.row0[i + 1] - row0;
    if (row >= tokens * a.group || tokens * a.group < a.rows_from || tokens * a.group > a.rows_to) return;
    const int64_t slot = (((int64_t)i * a.l.kv_heads + head) * a.max_rows + row) * a.splits;
    const int first = a.step.len[i] - tokens;
    const int t0 = row / a.row_tile * a.row_tile, t1 = min(tokens * a.group, t0 + a.row_tile) - 1;
    const int ranges = kv_ranges(kv_tiles(first + t0 / a.group, first + t1 / a.group, a.window, a.sinks).count(), a);
    const int width = D / 4, groups = 256 / width, group = tid / width, c = tid - group * width;
    const float4 *part = (const float4 *)(a.part + slot * D) + c;
    float4 ahead[kAhead];
    const bool works = group < groups;
#pragma unroll
    for (int j = 0; j < kAhead; j++) {
        const int s = group + j * groups;
        if (works && s < ranges) ahead[j] = part[(int64_t)s * width];
    }
    float m = -__builtin_inff(), l = 0.0f;
    if (tid < ranges) {
        const float2 ml = *(const float2 *)(a.part_ml + 2 * (slot + tid));
        m = ml.x, l = ml.y;
    }
    float most = m;
    for (int d = 32; d; d >>= 1) most = fmaxf(most, __shfl_xor(most, d));
    if ((tid & 63) == 0) red[0][tid >> 6] = most;
    __syncthreads();
    most = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
    const float f = most > -__builtin_inff() ? __builtin_amdgcn_exp2f(m - most) : 1.0f;  // of no visible token: sums of 0, or NaN
    fs[tid] = f;
    l *= f;
    if (tid >= ranges) l = 0.0f;
    for (int d = 32; d; d >>= 1) l += __shfl_xor(l, d);
    if ((tid & 63) == 0) red[1][tid >> 6] = l;
    __syncthreads();
    const float total = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    auto add = [&](const float4 &p, float by) {
        sum.x = __builtin_fmaf(p.x, by, sum.x), sum.y = __builtin_fmaf(p.y, by, sum.y);
        sum.z = __builtin_fmaf(p.z, by, sum.z), sum.w = __builtin_fmaf(p.w, by, sum.w);
    };
    if (works) {
#pragma unroll
        for (int j = 0; j < kAhead; j++) {
            const int s = group + j * groups;
            if (s < ranges) add(ahead[j], fs[s]);
        }
        for (int s = group + kAhead * groups; s < ranges; s += groups) add(part[(int64_t)s * width], fs[s]);
    }
    sums[tid] = sum;
    __syncthreads();
    if (tid >= width) return;
    for (int g = 1; g < groups; g++) add(sums[tid + g * width], 1.0f);
    const int64_t to = (int64_t)(row0 + row / a.group) * a.out_stride + (head * a.group + row % a.group) * D + 4 * c;
    const float by = total == 0.0f ? 0.0f : 1.0f / total;
    store_out(a.out, to, a.out_bf16, sum.x * by);
    store_out(a.out, to + 1, a.out_bf16, sum.y * by);
    store_out(a.out, to + 2, a.out_bf16, sum.z * by);
    store_out(a.out, to + 3, a.out_bf16, sum.w * by);
}

// The same for at most kFewRanges ranges: D / 4 threads a row, all of whose parts are on their way at once.
constexpr int kFewRanges = 16;
__global__ void __launch_bounds__(256) join_few_kernel(KvAttend a) {
    const int i = blockIdx.z, head = blockIdx.y, D = a.l.dim, width = D / 4, rows = 256 / width;
    const int group = threadIdx.x / width, c = threadIdx.x - group * width, row = blockIdx.x * rows + group;
    const int row0 = a.step.row0[i], tokens = a.step.row0[i + 1] - row0;
    if (group >= rows || row >= tokens * a.group || tokens * a.group < a.rows_from || tokens * a.group > a.rows_to) return;
    const int64_t slot = (((int64_t)i * a.l.kv_heads + head) * a.max_rows + row) * a.splits;
    const int first = a.step.len[i] - tokens;
    const int t0 = row / a.row_tile * a.row_tile, t1 = min(tokens * a.group, t0 + a.row_tile) - 1;
    const int ranges = kv_ranges(kv_tiles(first + t0 / a.group, first + t1 / a.group, a.window, a.sinks).count(), a);
    const float4 *part = (const float4 *)(a.part + slot * D) + c;
    const float2 *ml = (const float2 *)(a.part_ml + 2 * slot);
    float4 p[kFewRanges];
    float2 m[kFewRanges];
#pragma unroll
    for (int s = 0; s < kFewRanges; s++)
        if (s < ranges) p[s] = part[(int64_t)s * width], m[s] = ml[s];
    float most = -__builtin_inff();
#pragma unroll
    for (int s = 0; s < kFewRanges; s++)
        if (s < ranges) most = fmaxf(most, m[s].x);
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float total = 0.0f;
#pragma unroll
    for (int s = 0; s < kFewRanges; s++)
        if (s < ranges) {
            const float f = most > -__builtin_inff() ? __builtin_amdgcn_exp2f(m[s].x - most) : 1.0f;  // of no visible token: sums of 0, or NaN
            total = __builtin_fmaf(m[s].y, f, total);
            sum.x = __builtin_fmaf(p[s].x, f, sum.x), sum.y = __builtin_fmaf(p[s].y, f, sum.y);
            sum.z = __builtin_fmaf(p[s].z, f, sum.z), sum.w = __builtin_fmaf(p[s].w, f, sum.w);
        }
    const int64_t to = (int64_t)(row0 + row / a.group) * a.out_stride + (head * a.group + row % a.group) * D + 4 * c;
    const float by = total == 0.0f ? 0.0f : 1.0f / total;
    store_out(a.out, to, a.out_bf16, sum.x * by);
    store_out(a.out, to + 1, a.out_bf16, sum.y * by);
    store_out(a.out, to + 2, a.out_bf16, sum.z * by);
    store_out(a.out, to + 3, a.out_bf16, sum.w * by);
}

template <int R>
hipError_t decode(const KvAttend &a, hipStream_t s, hipEvent_t done) {
    const dim3 grid((unsigned)a.splits, (unsigned)(a.l.kv_heads * ((a.max_rows + R - 1) / R)), (unsigned)a.step.n);
    switch (a.l.dim) {
    case 64: return launch_with_event(decode_kernel<64, R>, grid, dim3(64 * waves_of(64)), s, done, a);
    case 96: return launch_with_event(decode_kernel<96, R>, grid, dim3(64 * waves_of(96)), s, done, a);
    case 128: return launch_with_event(decode_kernel<128, R>, grid, dim3(64 * waves_of(128)), s, done, a);
    case 192: return launch_with_event(decode_kernel<192, R>, grid, dim3(64 * waves_of(192)), s, done, a);
    case 256: return launch_with_event(decode_kernel<256, R>, grid, dim3(64 * waves_of(256)), s, done, a);
    }
    return hipErrorInvalidValue;
}

}  // namespace

hipError_t launch_kv_decode(const KvAttend &a, hipStream_t s, hipEvent_t done) {
    hipEvent_t last = a.splits > 1 ? nullptr : done;
    const hipError_t e = a.row_tile == 4 ? decode<4>(a, s, last) : decode<8>(a, s, last);
    return e == hipSuccess && a.splits > 1 ? launch_kv_join(a, s, done) : e;
}

hipError_t launch_kv_join(const KvAttend &a, hipStream_t s, hipEvent_t done) {
    if (a.splits <= kFewRanges) {
        const int rows = 256 / (a.l.dim / 4);
        return launch_with_event(join_few_kernel, dim3((unsigned)((a.max_rows + rows - 1) / rows), (unsigned)a.l.kv_heads, (unsigned)a.step.n), dim3(256), s, done, a);
    }
    return launch_with_event(join_kernel, dim3((unsigned)a.max_rows, (unsigned)a.l.kv_heads, (unsigned)a.step.n), dim3(256), s, done, a);
}

}  // namespace j4q
