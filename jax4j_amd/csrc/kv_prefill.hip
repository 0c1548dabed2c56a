// Attention over the 8-bit cache where a sequence has many query rows (prompts, chunks of them): 128 or 256 rows (tokens x query
// heads of a kv head) per workgroup against tiles of 64 tokens, bound by the matrix cores and the softmax between them.
//
// The formula is that of kv_decode.hip (the value scale inside the exponent). Here codes become fp16 (exact), once per
// workgroup and tile, on the way into LDS, and both products run on the fp16 matrix instruction 32x32x16 with fp32 sums:
//   scores   C[token][row]   = K[token][channel] q[channel][row]
//   output   C[channel][row] += V[channel][token] w[token][row]
// A lane has column (row) l % 32 of C, so maxima, sums and rescaling are its own but for the lane across (l ^ 32). It holds
// tokens 8 (r / 4) + 4 (l / 32) + r % 4 of a score product: they become its half of the second operand of two output steps as
// they are, since V's tokens lie in LDS in that order.
// q (scaled by a power of two per row) and w in fp16 round by 2^-11, which a bf16 result hides; for an fp32 result both are a sum
// of two fp16 (22 bits), twice the matrix instructions.
// m moves only when a t passes it by 7 octaves (w < 2^15 then), so the outputs are rescaled rarely.
//
// 8 kv heads of 128, 32 query heads, a prompt of 8192 into bf16: 553 to 600 us (from one card to another), 917 to 994 TFLOP/s, 67
// to 72 % of a plain matrix product's rate. Matrix instructions take 48 % of the SIMDs' cycles and vector ones 52 %: of
// two waves on a SIMD they add, whether or not they are brought side by side (half a round apart, with a barrier more:
// 2 % slower). Per tile and wave 32 of the first, 210 of the others: 32 exponentials, as many scalings, maxima (16, of three),
// sums, 16 roundings, 40 for the wave's share of the conversion. Without the fences 2.3 % slower.
#include <type_traits>

#include "kv.h"

// Nothing is scheduled across.
#define FENCE() __builtin_amdgcn_sched_barrier(0)

namespace j4q {
namespace {

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef __bf16 v4b __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef int v4i __attribute__((ext_vector_type(4)));
typedef int v16i __attribute__((ext_vector_type(16)));

constexpr float kUnit = 8.0f;  // the weight of t = m: 2^8
constexpr float kHead = 7.0f;

struct Two {
    float a, b;
};
// Own value and that of lane ^ 32, in either order. The empty asm keeps the compiler from taking the two results for one.
__device__ __forceinline__ Two swap32(float v) {
    uint32_t x = __builtin_bit_cast(uint32_t, v), y = x;
    asm("" : "+v"(y));
    const auto r = __builtin_amdgcn_permlane32_swap(x, y, false, false);
    return {__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1])};
}
__device__ __forceinline__ float max32(float v) {
    const Two t = swap32(v);
    return fmaxf(t.a, t.b);
}

// Four int8 codes as fp16: 1024 + 128 + code is exact in fp16, and so is the difference.
__device__ __forceinline__ void codes_to_half(uint32_t c, uint32_t *out) {
    const uint32_t u = c ^ 0x80808080u;
    const v2h bias = {(_Float16)1152.0f, (_Float16)1152.0f};
    out[0] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) - bias);
    out[1] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) - bias);
}

// 8 values from i on, 16-byte aligned.
__device__ __forceinline__ void load8(const void *p, int64_t i, int bf16, float *x) {
    if (bf16) {
        const uint4 t = *(const uint4 *)((const uint16_t *)p + i);
        const uint32_t w[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
        for (int j = 0; j < 4; j++) {
            x[2 * j] = __builtin_bit_cast(float, w[j] << 16);
            x[2 * j + 1] = __builtin_bit_cast(float, w[j] & 0xffff0000u);
        }
    } else {
        const float4 *from = (const float4 *)((const float *)p + i);
        const float4 t = from[0], u = from[1];
        x[0] = t.x, x[1] = t.y, x[2] = t.z, x[3] = t.w, x[4] = u.x, x[5] = u.y, x[6] = u.z, x[7] = u.w;
    }
}
// W: waves, of 32 rows each. P: fp16 parts of q and w, 1 for a bf16 result, 2 for an fp32 one.
template <int D, int W, int P>
__global__ void __launch_bounds__(64 * W, D <= 128 ? 2 : 1) prefill_kernel(KvAttend a) {
    constexpr int kThreads = 64 * W, kRows = 32 * W;
    constexpr int KP = D + 8, VP = kKvTile + 8;            // row pitches in LDS: an odd number of 16 bytes, 16 rows on all banks
    constexpr int N = (4 * D + kThreads - 1) / kThreads;   // 16-byte pieces of K, and of V, that a thread stages
    __shared__ __align__(16) _Float16 ks[2][kKvTile][KP];
    __shared__ __align__(16) _Float16 vs[2][D][VP];
    __shared__ __align__(16) float scales[2][3][4];        // K scale, log2 of V's, its reciprocal
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 31, half = lane >> 5;
    const int head = blockIdx.x % a.l.kv_heads, split = blockIdx.x / a.l.kv_heads, i = blockIdx.z;
    const int row0 = a.step.row0[i], tokens = a.step.row0[i + 1] - row0, len = a.step.len[i], rows = tokens * a.group;
    const int tile_count = (rows + kRows - 1) / kRows;
    if ((int)blockIdx.y >= tile_count || rows < a.rows_from) return;
    const int r0 = (tile_count - 1 - (int)blockIdx.y) * kRows;  // the longest first
    const int r1 = min(rows, r0 + kRows) - 1;
    const int before = len - tokens;
    const KvTiles vis = kv_tiles(before + r0 / a.group, before + r1 / a.group, a.window, a.sinks);
    int t0 = 0, t1 = vis.count();
    if (a.splits > 1) {
        const int each = kv_range_tiles(t1, a);
        t0 = split * each;
        if (t0 >= t1) return;
        t1 = min(t1, t0 + each);
    }
    // the wave's rows, and its places; the lane's row
    const int w0 = r0 + wave * 32, w1 = min(r1, w0 + 31);
    const int p_first = before + min(w0, r1) / a.group, p_last = before + w1 / a.group;
    const int row = min(w0 + col, r1), place = before + row / a.group;
    v8h q[P][D / 16];
    float qk;
    {
        const int64_t at = (int64_t)(row0 + row / a.group) * a.q_stride + (head * a.group + row % a.group) * D + 8 * half;
        float x[D / 16][8], most = 0.0f, finite = 0.0f;
#pragma unroll
        for (int s = 0; s < D / 16; s++) load8(a.q, at + 16 * s, a.q_bf16, x[s]);
#pragma unroll
        for (int s = 0; s < D / 16; s++)
#pragma unroll
            for (int j = 0; j < 8; j++) {
                most = fmaxf(most, fabsf(x[s][j]));
                finite = __builtin_fmaf(x[s][j], 0.0f, finite);  // else NaN
            }
        most = max32(most);
        const Two both = swap32(finite);
        // to [2^13, 2^14), by a power of two (2^100 at most)
        const int e = max((int)(__builtin_bit_cast(uint32_t, most) >> 23) - 127 - 13, -100);
        const float up = __builtin_bit_cast(float, (uint32_t)(127 - e) << 23);
        qk = __builtin_bit_cast(float, (uint32_t)(127 + e) << 23) * a.scale + (both.a + both.b);
#pragma unroll
        for (int s = 0; s < D / 16; s++)
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float y = x[s][j] * up;
                q[0][s][j] = (_Float16)y;
                if constexpr (P == 2) q[1][s][j] = (_Float16)(y - (float)q[0][s][j]);
            }
    }

    v16f o[D / 32];
#pragma unroll
    for (int d = 0; d < D / 32; d++)
#pragma unroll
        for (int r = 0; r < 16; r++) o[d][r] = 0.0f;
    // lim: the t (less m) that is too large
    float m_at = -__builtin_inff(), base = 0.0f, lim = -__builtin_inff(), l_sum = 0.0f;

    const int32_t *table = a.step.table + (int64_t)a.step.seq[i] * a.step.sequence_pages;
    const int last_block = (len - 1) / kKvBlock, in_mask = (1 << a.l.block_shift) - 1;
    // Piece c of K and of V lies 16 (c % D) bytes into that of block c / D, which is the same for a wave where 64 divides D. Pages
    // are looked up a tile ahead of the loads from them, those a tile ahead of their conversion.
    int page[N], scale_page;
    uint4 kraw[N], vraw[N];
    float2 sraw = make_float2(0.0f, 0.0f);
    auto block_of = [&](int j) { return D % 64 == 0 ? __builtin_amdgcn_readfirstlane((tid + kThreads * j) / D) : (tid + kThreads * j) / D; };
    auto staged = [&](int j) { return 4 * D % kThreads == 0 || tid + kThreads * j < 4 * D; };
    auto look_up = [&](int tile) {
#pragma unroll
        for (int j = 0; j < N; j++)
            if (staged(j)) page[j] = table[min(tile * 4 + block_of(j), last_block) >> a.l.block_shift];
        if (wave == 0) scale_page = table[min(tile * 4 + (lane & 3), last_block) >> a.l.block_shift];
    };
    auto fetch = [&](int tile) {
#pragma unroll
        for (int j = 0; j < N; j++) {
            if (!staged(j)) continue;
            const int blk = min(tile * 4 + block_of(j), last_block), in = (head << a.l.block_shift) + (blk & in_mask);
            const int pg = D % 64 == 0 ? __builtin_amdgcn_readfirstlane(page[j]) : page[j];
            const uint8_t *k = a.l.base + (int64_t)max(pg, 0) * a.l.page_bytes + in * (2 * kKvBlock * D);
            const int at = (tid + kThreads * j) % D * 16;
            kraw[j] = *(const uint4 *)(k + at);
            vraw[j] = *(const uint4 *)(k + kKvBlock * D + at);
        }
        if (wave != 0) return;
        const int blk = min(tile * 4 + (lane & 3), last_block), in = (head << a.l.block_shift) + (blk & in_mask);
        sraw = *(const float2 *)(a.l.base + (int64_t)max(scale_page, 0) * a.l.page_bytes + a.l.scales + 8 * in);
    };
    // a quarter of a pair of pieces: 8 codes of K (units 0, 1) or V (2, 3) to LDS
    auto stage_unit = [&](int buf, int unit) {
        const int j = unit / 4, c = tid + kThreads * j;
        if (!staged(j)) return;
        uint32_t h[4];
        if (unit % 4 < 2) {
            codes_to_half(unit % 2 ? kraw[j].z : kraw[j].x, h), codes_to_half(unit % 2 ? kraw[j].w : kraw[j].y, h + 2);
            *(uint4 *)&ks[buf][c / (D / 16)][c % (D / 16) * 16 + unit % 2 * 8] = make_uint4(h[0], h[1], h[2], h[3]);
        } else {
            codes_to_half(unit % 2 ? vraw[j].y : vraw[j].x, h), codes_to_half(unit % 2 ? vraw[j].w : vraw[j].z, h + 2);
            *(uint4 *)&vs[buf][c % D][c / D * 16 + unit % 2 * 8] = make_uint4(h[0], h[1], h[2], h[3]);
        }
    };
    auto stage_scales = [&](int buf) {
        if (wave != 0) return;
        // what lies behind the end is hidden, and must only not be NaN
        const bool nan = sraw.y != sraw.y;
        const float sv = nan ? 1.0f : fmaxf(sraw.y, kKvMinScale);
        if (lane < 4) {
            scales[buf][0][lane] = sraw.x;
            scales[buf][1][lane] = nan ? sraw.y : __builtin_amdgcn_logf(sv);
            scales[buf][2][lane] = __builtin_amdgcn_rcpf(sv);
        }
    };

    // behind the last tile the last one again, which nobody uses: no branch inside the round
    auto tile_at = [&](int u) { return vis.tile(min(u, t1 - 1)); };
    if (t0 < t1) {
        look_up(tile_at(t0));
        fetch(tile_at(t0));
        look_up(tile_at(t0 + 1));
        for (int unit = 0; unit < 4 * N; unit++) stage_unit(0, unit);
        stage_scales(0);
        fetch(tile_at(t0 + 1));
        look_up(tile_at(t0 + 2));
    }
    __syncthreads();
    // One tile. The order is that of the source (the fences): each product goes with vector work that does not wait for it, the
    // next tile's conversion beside the first half of the scores, their first half's scaling beside the second, and each
    // block's weights beside the output products of the block before.
    auto round = [&](int u, auto masked) {
        constexpr int G = D / 16, E = D / 32, kAhead = 8, vAhead = 8;  // operands on their way from LDS
        constexpr bool kMasked = decltype(masked)::value;
        const int buf = (u - t0) & 1, j0 = vis.tile(u) * kKvTile;
        v16f s[2];
        v8h k[kAhead], v[vAhead];
        float t[2][16], top[2] = {-__builtin_inff(), -__builtin_inff()};
        float f[4], c[4], rsv[4];
#pragma unroll
        for (int r = 0; r < 16; r++) s[0][r] = s[1][r] = 0.0f;
        auto scores = [&](int sub, int st) {
#pragma unroll
            for (int p = 0; p < P; p++) s[sub] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k[(sub * G + st) % kAhead], q[p][st], s[sub], 0, 0, 0);
        };
        auto scaled = [&](int sub, int r) {
            float x = __builtin_fmaf(s[sub][r], f[2 * sub + r / 8], c[2 * sub + r / 8]);
            if constexpr (kMasked) {
                const int at = j0 + 32 * sub + 8 * (r / 4) + 4 * half + r % 4;
                const bool seen = (at <= place) & ((at > place - a.window) | (at < a.sinks));
                x = seen ? x : -__builtin_inff();
            }
            t[sub][r] = x;
            top[sub] = fmaxf(top[sub], x);
        };
        auto read_k = [&](int n) {
            if (n < 2 * G) k[n % kAhead] = *(const v8h *)&ks[buf][32 * (n / G) + col][16 * (n % G) + 8 * half];
        };
        auto read_v = [&](int n) {
            if (n < 4 * E) v[n % vAhead] = *(const v8h *)&vs[buf][32 * (n % E) + col][16 * (n / E) + 8 * half];
        };

#pragma unroll
        for (int n = 0; n < kAhead; n++) read_k(n);
        FENCE();
#pragma unroll
        for (int st = 0; st < G; st++) {
            scores(0, st);
            read_k(st + kAhead);
#pragma unroll
            for (int unit = st * 4 * N / G; unit < (st + 1) * 4 * N / G; unit++) stage_unit(buf ^ 1, unit);
            FENCE();
        }
        stage_scales(buf ^ 1);
#pragma unroll
        for (int b = 0; b < 4; b++) f[b] = qk * scales[buf][0][b], c[b] = scales[buf][1][b] + base, rsv[b] = scales[buf][2][b];
        fetch(tile_at(u + 2));
#pragma unroll
        for (int st = 0; st < G; st++) {
            scores(1, st);
            read_k(G + st + kAhead);
#pragma unroll
            for (int r = st * 16 / G; r < (st + 1) * 16 / G; r++) scaled(0, r);
            if (st == G - 2) {
#pragma unroll
                for (int n = 0; n < vAhead; n++) read_v(n);
            }
            FENCE();
        }
        look_up(tile_at(u + 3));
#pragma unroll
        for (int r = 0; r < 16; r++) scaled(1, r);
        float most = fmaxf(top[0], top[1]);
        if (__any(most > lim)) {
            most = max32(most);
            if (most > lim) {  // m moves up to the largest t: by `up` octaves
                const bool first = !(m_at > -__builtin_inff());
                const float up = first ? most : most - kUnit, shrink = first ? 0.0f : __builtin_amdgcn_exp2f(-up);
                m_at = first ? up : m_at + up;
                const float shift = kUnit - m_at - base;
                base = kUnit - m_at;
                lim = kUnit + kHead;
                l_sum *= shrink;
#pragma unroll
                for (int r = 0; r < 32; r++) t[r / 16][r % 16] += shift;
#pragma unroll
                for (int d = 0; d < E; d++)
#pragma unroll
                    for (int r = 0; r < 16; r++) o[d][r] *= shrink;
            }
        }
        // The sum is of the weights before they are rounded: where a block's value scale is far below others', its weights may fall
        // below what fp16 holds, and count in the sum all the same.
        v8h w[2][P];
        float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        auto weights = [&](int b, int r) {
            const float e0 = __builtin_amdgcn_exp2f(t[b / 2][b % 2 * 8 + r]), e1 = __builtin_amdgcn_exp2f(t[b / 2][b % 2 * 8 + r + 1]);
            const v2h h = {(_Float16)e0, (_Float16)e1};
            w[b % 2][0][r] = h[0], w[b % 2][0][r + 1] = h[1];
            if constexpr (P == 2) w[b % 2][1][r] = (_Float16)(e0 - (float)h[0]), w[b % 2][1][r + 1] = (_Float16)(e1 - (float)h[1]);
            sum[b] += e0 + e1;
        };
#pragma unroll
        for (int r = 0; r < 8; r += 2) weights(0, r);
        FENCE();
#pragma unroll
        for (int b = 0; b < 4; b++) {
#pragma unroll
            for (int d = 0; d < E; d++) {
#pragma unroll
                for (int p = 0; p < P; p++) o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[(b * E + d) % vAhead], w[b % 2][p], o[d], 0, 0, 0);
                read_v(b * E + d + vAhead);
                if (b < 3) {
#pragma unroll
                    for (int r = d * 4 / E; r < (d + 1) * 4 / E; r++) weights(b + 1, 2 * r);
                }
                FENCE();
            }
            l_sum = __builtin_fmaf(sum[b], rsv[b], l_sum);
        }
        __syncthreads();
    };
    // a tile of which every row of the wave sees every token
    auto whole = [&](int u) {
        const int j0 = vis.tile(u) * kKvTile, j1 = j0 + kKvTile - 1;
        return j1 <= p_first && (j0 > p_last - a.window || j1 < a.sinks);
    };
    // a wave without rows stages its share of the tiles and no more (32 rows of 128: 510 us, 220 so)
    if (w0 > r1)
        for (int u = t0; u < t1; u++) {
            const int buf = (u - t0) & 1;
#pragma unroll
            for (int unit = 0; unit < 4 * N; unit++) stage_unit(buf ^ 1, unit);
            fetch(tile_at(u + 2));
            look_up(tile_at(u + 3));
            __syncthreads();
        }
    for (int u = w0 > r1 ? t1 : t0; u < t1;) {
        for (; u < t1 && whole(u); u++) round(u, std::false_type());
        for (; u < t1 && !whole(u); u++) round(u, std::true_type());
    }

    const int r = w0 + col;
    const Two both = swap32(l_sum);
    const float total = both.a + both.b;
    if (r > r1) return;
    if (a.splits > 1) {
        const int64_t slot = (((int64_t)i * a.l.kv_heads + head) * a.max_rows + r) * a.splits + split;
#pragma unroll
        for (int d = 0; d < D / 32; d++)
#pragma unroll
            for (int g = 0; g < 4; g++)
                *(float4 *)(a.part + slot * D + 32 * d + 8 * g + 4 * half) = make_float4(o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]);
        if (half == 0) {
            a.part_ml[2 * slot] = m_at;
            a.part_ml[2 * slot + 1] = total;
        }
    } else {
        const float f = total == 0.0f ? 0.0f : 1.0f / total;
        const int64_t to = (int64_t)(row0 + r / a.group) * a.out_stride + (head * a.group + r % a.group) * D + 4 * half;
#pragma unroll
        for (int d = 0; d < D / 32; d++)
#pragma unroll
            for (int g = 0; g < 4; g++) {
                const float4 x = make_float4(o[d][4 * g] * f, o[d][4 * g + 1] * f, o[d][4 * g + 2] * f, o[d][4 * g + 3] * f);
                const int64_t at = to + 32 * d + 8 * g;
                if constexpr (P == 1) *(v4b *)((uint16_t *)a.out + at) = v4b{(__bf16)x.x, (__bf16)x.y, (__bf16)x.z, (__bf16)x.w};
                else *(float4 *)((float *)a.out + at) = x;
            }
    }
}

// The same for up to 32 rows, where memory is the bound: a wave walks tiles of its own, as in kv_decode.hip, loaded a tile ahead, and
// nothing goes through LDS but the last sum. What it loads is the operands as they are: 16 channels of a key, for the int8
// instruction 32x32x32, and 16 tokens of a value channel, converted to fp16 for two steps of 32x32x16. Row m of a score product
// is token 16 (m / 4 % 2) + 4 (m / 8) + m % 4, so that a lane's 16 scores are those of block l / 32 in order.
// q enters as whole numbers over its row's largest magnitude, in digits to the base 256: two (16 bits) for a bf16 result, three
// (24) for an fp32 one. Values enter as the codes that they are: with a bias that is taken off in the end (three instructions for
// four codes instead of five) every weight's rounding counts 128 times in every channel, however small its codes.
// 8 kv heads of 128, 64 sequences of 8000 tokens (1.05 GB), 20 rows: 178 us into bf16, 5.9 TB/s, and 200 fp32; the kernel above
// took 510 and 787. Pages looked up behind the loads of a tile, or a branch around these, let the compiler wait for them (117
// us instead of 104, heads of 64); the conversion of keys to fp16 made it 272 fp32.
template <int D, int P>
__global__ void __launch_bounds__(512, 2) rows_kernel(KvAttend a) {
    constexpr int W = 8, S = D / 32;         // waves; pieces of 16 channels that a lane has of a key, and blocks of 32 value channels
    constexpr int kPitch = D + 4;
    __shared__ __align__(16) float part[W][32][kPitch];
    __shared__ float part_ml[W][32][2];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 31, half = lane >> 5;
    const int i = blockIdx.z, head = blockIdx.y % a.l.kv_heads, rg = blockIdx.y / a.l.kv_heads;
    const int row0 = a.step.row0[i], tokens = a.step.row0[i + 1] - row0, len = a.step.len[i], rows = tokens * a.group;
    const int r0 = rg * 32, r1 = min(rows, r0 + 32) - 1;
    if (r0 >= rows || rows < a.rows_from || rows > a.rows_to) return;
    const int before = len - tokens;
    const KvTiles vis = kv_tiles(before + r0 / a.group, before + r1 / a.group, a.window, a.sinks);
    int t0 = 0, t1 = vis.count();
    if (a.splits > 1) {
        const int each = kv_range_tiles(t1, a);
        t0 = blockIdx.x * each;
        if (t0 >= t1) return;
        t1 = min(t1, t0 + each);
    }
    const int p_first = before + r0 / a.group, p_last = before + r1 / a.group;
    const int row = min(r0 + col, r1), place = before + row / a.group;

    const int32_t *table = a.step.table + (int64_t)a.step.seq[i] * a.step.sequence_pages;
    const int last_block = (len - 1) / kKvBlock, in_mask = (1 << a.l.block_shift) - 1;
    const int k_block = col >> 2 & 1, k_token = 4 * (col >> 3) + (col & 3);
    v4i kraw[2][S];
    uint4 vraw[2][S];
    float2 sraw[2];
    // Pages are looked up before the loads of the tile in front of theirs: a wait for them is none for those.
    struct Pages {
        int k[2], v[2];
    } pages;
    auto look_up = [&](int tile) {
        Pages p;
#pragma unroll
        for (int sub = 0; sub < 2; sub++) {
            p.k[sub] = table[min(tile * 4 + 2 * sub + k_block, last_block) >> a.l.block_shift];
            p.v[sub] = table[min(tile * 4 + 2 * sub + half, last_block) >> a.l.block_shift];
        }
        return p;
    };
    // A page that is not there gives bytes that weigh nothing.
    auto block_at = [&](int block, int page, int *in) {
        *in = (head << a.l.block_shift) + (min(block, last_block) & in_mask);
        return a.l.base + (int64_t)max(page, 0) * a.l.page_bytes;
    };
    auto fetch_k = [&](int tile, int sub, const Pages &p) {
        int in;
        const uint8_t *pg = block_at(tile * 4 + 2 * sub + k_block, p.k[sub], &in), *k = pg + in * (2 * kKvBlock * D) + k_token * D + half * 16;
#pragma unroll
        for (int s = 0; s < S; s++) kraw[sub][s] = *(const v4i *)(k + 32 * s);
    };
    auto fetch_v = [&](int tile, int sub, const Pages &p) {
        int in;
        const uint8_t *pg = block_at(tile * 4 + 2 * sub + half, p.v[sub], &in), *v = pg + in * (2 * kKvBlock * D) + kKvBlock * D + col * 16;
        sraw[sub] = *(const float2 *)(pg + a.l.scales + 8 * in);
#pragma unroll
        for (int d = 0; d < S; d++) vraw[sub][d] = *(const uint4 *)(v + 512 * d);
    };
    if (t0 + wave < t1) {
        const int tile = vis.tile(t0 + wave);
        const Pages first = look_up(tile);
        pages = look_up(vis.tile(min(t0 + wave + W, t1 - 1)));
#pragma unroll
        for (int sub = 0; sub < 2; sub++) {
            fetch_k(tile, sub, first);
            fetch_v(tile, sub, first);
        }
    }

    constexpr int kDigits = P + 1;
    constexpr float kMost = P == 1 ? 32600.0f : 8355000.0f;  // what the digits hold, and room for rounding
    v4i q[kDigits][S];                                       // the lowest first
    float qk;
    {
        const int64_t at = (int64_t)(row0 + row / a.group) * a.q_stride + (head * a.group + row % a.group) * D + 16 * half;
        float x[S][16], most = 0.0f, finite = 0.0f;
#pragma unroll
        for (int s = 0; s < S; s++) {
            load8(a.q, at + 32 * s, a.q_bf16, x[s]);
            load8(a.q, at + 32 * s + 8, a.q_bf16, x[s] + 8);
#pragma unroll
            for (int j = 0; j < 16; j++) {
                most = fmaxf(most, fabsf(x[s][j]));
                finite = __builtin_fmaf(x[s][j], 0.0f, finite);  // else NaN
            }
        }
        const Two both = swap32(finite);
        // at least 2^-90, so that its reciprocal is finite
        const float unit = fmaxf(max32(most), 0x1p-90f) / kMost, inv = 1.0f / unit;
        qk = unit * a.scale + (both.a + both.b);
#pragma unroll
        for (int s = 0; s < S; s++)
#pragma unroll
            for (int n = 0; n < 4; n++) {
                uint32_t v[4];
#pragma unroll
                for (int j = 0; j < 4; j++) v[j] = ((uint32_t)(int)rintf(x[s][4 * n + j] * inv) + 0x808080u) ^ 0x808080u;
#pragma unroll
                for (int g = 0; g < kDigits; g++) {
                    uint32_t w = 0;
#pragma unroll
                    for (int j = 0; j < 4; j++) w |= (v[j] >> (8 * g) & 0xffu) << (8 * j);
                    q[g][s][n] = (int)w;
                }
            }
    }

    v16f o[S];
#pragma unroll
    for (int d = 0; d < S; d++)
#pragma unroll
        for (int r = 0; r < 16; r++) o[d][r] = 0.0f;
    float m_at = -__builtin_inff(), base = 0.0f, lim = -__builtin_inff(), l_sum = 0.0f;
    auto halves = [&](uint32_t c0, uint32_t c1) {
        uint32_t h[4];
        codes_to_half(c0, h), codes_to_half(c1, h + 2);
        return __builtin_bit_cast(v8h, make_uint4(h[0], h[1], h[2], h[3]));
    };
    // One tile. The last one's round is another, since with a branch round the loads of the next the compiler waits for all of them.
    auto round = [&](int u, auto more) {
        constexpr bool kMore = decltype(more)::value;
        const int tile = vis.tile(u), next = vis.tile(min(u + W, t1 - 1)), j0 = tile * kKvTile, j1 = j0 + kKvTile - 1;
        const Pages at_next = pages;
        if constexpr (kMore) pages = look_up(vis.tile(min(u + 2 * W, t1 - 1)));
        const bool masked = !(j1 <= p_first && (j0 > p_last - a.window || j1 < a.sinks));
#pragma unroll
        for (int sub = 0; sub < 2; sub++) {
            v16i high, low;
            v16f t;
#pragma unroll
            for (int r = 0; r < 16; r++) high[r] = low[r] = 0;
#pragma unroll
            for (int s = 0; s < S; s++) high = __builtin_amdgcn_mfma_i32_32x32x32_i8(kraw[sub][s], q[kDigits - 1][s], high, 0, 0, 0);
            if constexpr (P == 2) {
#pragma unroll
                for (int s = 0; s < S; s++) low = __builtin_amdgcn_mfma_i32_32x32x32_i8(kraw[sub][s], q[0][s], low, 0, 0, 0);
            }
#pragma unroll
            for (int r = 0; r < 16; r++) high[r] *= 256;
#pragma unroll
            for (int s = 0; s < S; s++) high = __builtin_amdgcn_mfma_i32_32x32x32_i8(kraw[sub][s], q[kDigits - 2][s], high, 0, 0, 0);
            if constexpr (kMore) fetch_k(next, sub, at_next);
            const bool nan = sraw[sub].y != sraw[sub].y;
            const float sv = nan ? 1.0f : fmaxf(sraw[sub].y, kKvMinScale), rsv = __builtin_amdgcn_rcpf(sv);
            const float f = qk * sraw[sub].x, c = (nan ? sraw[sub].y : __builtin_amdgcn_logf(sv)) + base;
            float most = -__builtin_inff();
#pragma unroll
            for (int r = 0; r < 16; r++) t[r] = __builtin_fmaf(P == 2 ? __builtin_fmaf((float)high[r], 256.0f, (float)low[r]) : (float)high[r], f, c);
            if (masked) {
                int at0 = j0 + 32 * sub + 16 * half;
                asm volatile("" : "+v"(at0));  // else the comparisons are made in front of the branch, for every tile
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    const int at = at0 + r;
                    const bool seen = (at <= place) & ((at > place - a.window) | (at < a.sinks));
                    t[r] = seen ? t[r] : -__builtin_inff();
                }
            }
#pragma unroll
            for (int r = 0; r < 16; r++) most = fmaxf(most, t[r]);
            if (__any(most > lim)) {
                most = max32(most);
                if (most > lim) {  // m moves up to the largest t
                    const bool first = !(m_at > -__builtin_inff());
                    const float up = first ? most : most - kUnit, shrink = first ? 0.0f : __builtin_amdgcn_exp2f(-up);
                    m_at = first ? up : m_at + up;
                    const float shift = kUnit - m_at - base;
                    base = kUnit - m_at;
                    lim = kUnit + kHead;
                    l_sum *= shrink;
#pragma unroll
                    for (int r = 0; r < 16; r++) t[r] += shift;
#pragma unroll
                    for (int d = 0; d < S; d++)
#pragma unroll
                        for (int r = 0; r < 16; r++) o[d][r] *= shrink;
                }
            }
            float sum = 0.0f;
            v8h w[P][2];
#pragma unroll
            for (int r = 0; r < 16; r++) {
                const float e = __builtin_amdgcn_exp2f(t[r]);
                const _Float16 h = (_Float16)e;
                w[0][r / 8][r % 8] = h;
                if constexpr (P == 2) w[1][r / 8][r % 8] = (_Float16)(e - (float)h);
                sum += e;
            }
            l_sum = __builtin_fmaf(sum, rsv, l_sum);
#pragma unroll
            for (int d = 0; d < S; d++) {
                const v8h v0 = halves(vraw[sub][d].x, vraw[sub][d].y), v1 = halves(vraw[sub][d].z, vraw[sub][d].w);
#pragma unroll
                for (int p = 0; p < P; p++) o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v0, w[p][0], o[d], 0, 0, 0);
#pragma unroll
                for (int p = 0; p < P; p++) o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v1, w[p][1], o[d], 0, 0, 0);
            }
            if constexpr (kMore) fetch_v(next, sub, at_next);
        }
    };
    int u = t0 + wave;
    for (; u + W < t1; u += W) round(u, std::true_type());
    if (u < t1) round(u, std::false_type());

    const Two both = swap32(l_sum);
#pragma unroll
    for (int d = 0; d < S; d++)
#pragma unroll
        for (int g = 0; g < 4; g++)
            *(float4 *)&part[wave][col][32 * d + 8 * g + 4 * half] = make_float4(o[d][4 * g], o[d][4 * g + 1], o[d][4 * g + 2], o[d][4 * g + 3]);
    if (half == 0) {
        part_ml[wave][col][0] = m_at;
        part_ml[wave][col][1] = both.a + both.b;
    }
    __syncthreads();
    for (int at = threadIdx.x; at < 32 * (D / 4); at += 512) {
        const int in = at / (D / 4), d = (at - in * (D / 4)) * 4, r = r0 + in;
        if (r > r1) break;
        float most = -__builtin_inff(), total = 0.0f;
        for (int w = 0; w < W; w++) most = fmaxf(most, part_ml[w][in][0]);
        float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int w = 0; w < W; w++) {
            const float f = most > -__builtin_inff() ? __builtin_amdgcn_exp2f(part_ml[w][in][0] - most) : 1.0f;
            const float4 x = *(const float4 *)&part[w][in][d];
            sum.x = __builtin_fmaf(x.x, f, sum.x), sum.y = __builtin_fmaf(x.y, f, sum.y);
            sum.z = __builtin_fmaf(x.z, f, sum.z), sum.w = __builtin_fmaf(x.w, f, sum.w);
            total = __builtin_fmaf(part_ml[w][in][1], f, total);
        }
        if (a.splits > 1) {
            const int64_t slot = (((int64_t)i * a.l.kv_heads + head) * a.max_rows + r) * a.splits + blockIdx.x;
            *(float4 *)(a.part + slot * D + d) = sum;
            if (d == 0) {
                a.part_ml[2 * slot] = most;
                a.part_ml[2 * slot + 1] = total;
            }
        } else {
            const float f = total == 0.0f ? 0.0f : 1.0f / total;
            const int64_t to = (int64_t)(row0 + r / a.group) * a.out_stride + (head * a.group + r % a.group) * D + d;
            if constexpr (P == 1) *(v4b *)((uint16_t *)a.out + to) = v4b{(__bf16)(sum.x * f), (__bf16)(sum.y * f), (__bf16)(sum.z * f), (__bf16)(sum.w * f)};
            else *(float4 *)((float *)a.out + to) = make_float4(sum.x * f, sum.y * f, sum.z * f, sum.w * f);
        }
    }
}

template <int W, int P>
hipError_t prefill(const KvAttend &a, hipStream_t s, hipEvent_t done) {
    const dim3 grid((unsigned)(a.l.kv_heads * a.splits), (unsigned)((a.max_rows + 32 * W - 1) / (32 * W)), (unsigned)a.step.n);
    switch (a.l.dim) {
    case 64: return launch_with_event(prefill_kernel<64, W, P>, grid, dim3(64 * W), s, done, a);
    case 96: return launch_with_event(prefill_kernel<96, W, P>, grid, dim3(64 * W), s, done, a);
    case 128: return launch_with_event(prefill_kernel<128, W, P>, grid, dim3(64 * W), s, done, a);
    case 192: return launch_with_event(prefill_kernel<192, 4, P>, grid, dim3(256), s, done, a);
    case 256: return launch_with_event(prefill_kernel<256, 4, P>, grid, dim3(256), s, done, a);
    }
    return hipErrorInvalidValue;
}

template <int D, int P>
hipError_t rows(const KvAttend &a, hipStream_t s, hipEvent_t done) {
    const dim3 grid((unsigned)a.splits, (unsigned)(a.l.kv_heads * ((a.max_rows + 31) / 32)), (unsigned)a.step.n);
    return launch_with_event(rows_kernel<D, P>, grid, dim3(512), s, done, a);
}

}  // namespace

hipError_t launch_kv_rows(const KvAttend &a, hipStream_t s, hipEvent_t done) {
    hipEvent_t last = a.splits > 1 ? nullptr : done;
    hipError_t e = hipErrorInvalidValue;
    switch (a.l.dim) {
    case 64: e = a.out_bf16 ? rows<64, 1>(a, s, last) : rows<64, 2>(a, s, last); break;
    case 96: e = a.out_bf16 ? rows<96, 1>(a, s, last) : rows<96, 2>(a, s, last); break;
    case 128: e = a.out_bf16 ? rows<128, 1>(a, s, last) : rows<128, 2>(a, s, last); break;
    }
    return e == hipSuccess && a.splits > 1 ? launch_kv_join(a, s, done) : e;
}

hipError_t launch_kv_prefill(const KvAttend &a, hipStream_t s, hipEvent_t done) {
    hipEvent_t last = a.splits > 1 ? nullptr : done;
    const bool wide = a.row_tile == 256;
    const hipError_t e = a.out_bf16 ? wide ? prefill<8, 1>(a, s, last) : prefill<4, 1>(a, s, last) : wide ? prefill<8, 2>(a, s, last) : prefill<4, 2>(a, s, last);
    return e == hipSuccess && a.splits > 1 ? launch_kv_join(a, s, done) : e;
}

}  // namespace j4q
