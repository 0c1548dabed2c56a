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
#include "kv.h"

namespace j4q {
namespace {

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef float v16f __attribute__((ext_vector_type(16)));

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

__device__ __forceinline__ float value_at(const void *p, int64_t i, int bf16) {
    return bf16 ? __builtin_bit_cast(float, (uint32_t)((const uint16_t *)p)[i] << 16) : ((const float *)p)[i];
}
__device__ __forceinline__ uint32_t bf16_bits(float f) {
    const uint32_t u = __builtin_bit_cast(uint32_t, f);
    return f != f ? (u >> 16) | 0x40 : (u + 0x7fffu + ((u >> 16) & 1)) >> 16;
}

// NT: tiles of 32 rows of a wave. P: fp16 parts of q and w.
template <int D, int NT, int P>
__global__ void __launch_bounds__(256, NT == 1 && D <= 128 ? 2 : 1) prefill_kernel(KvAttend a) {
    constexpr int kRows = 4 * NT * 32;
    constexpr int KP = D + 8, VP = kKvTile + 8;            // row pitches in LDS: an odd number of 16 bytes, 16 rows on all banks
    constexpr int N = (4 * D + 255) / 256;                 // 16-byte pieces of K, and of V, that a thread stages
    __shared__ __align__(16) _Float16 ks[2][kKvTile][KP];
    __shared__ __align__(16) _Float16 vs[2][D][VP];
    __shared__ __align__(16) float scales[2][3][4];        // K scale, log2 of V's, its reciprocal
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, col = lane & 31, half = lane >> 5;
    const int head = blockIdx.x % a.l.kv_heads, split = blockIdx.x / a.l.kv_heads, i = blockIdx.z;
    const int row0 = a.step.row0[i], tokens = a.step.row0[i + 1] - row0, len = a.step.len[i], rows = tokens * a.group;
    const int tile_count = (rows + kRows - 1) / kRows;
    if ((int)blockIdx.y >= tile_count) return;
    const int r0 = (tile_count - 1 - (int)blockIdx.y) * kRows;  // the longest first
    const int r1 = min(rows, r0 + kRows) - 1;
    const int before = len - tokens;
    const KvTiles vis = kv_tiles(before + r0 / a.group, before + r1 / a.group, a.window, a.sinks);
    int t0 = 0, t1 = vis.count();
    if (a.splits > 1) {
        const int ranges = kv_ranges(t1, a);
        if (split >= ranges) return;
        t0 = split * a.split_tiles;
        if (split + 1 < ranges) t1 = t0 + a.split_tiles;
    }
    // the wave's rows, and its places
    const int w0 = r0 + wave * NT * 32, w1 = min(r1, w0 + NT * 32 - 1);
    const int p_first = before + min(w0, r1) / a.group, p_last = before + w1 / a.group;
    int place[NT];
    v8h q[NT][P][D / 16];
    float qk[NT];
#pragma unroll
    for (int n = 0; n < NT; n++) {
        const int r = min(w0 + n * 32 + col, r1);
        place[n] = before + r / a.group;
        const int64_t at = (int64_t)(row0 + r / a.group) * a.q_stride + (head * a.group + r % a.group) * D + 8 * half;
        float most = 0.0f;
        for (int s = 0; s < D / 16; s++)
            for (int j = 0; j < 8; j++) {
                const float m = fabsf(value_at(a.q, at + 16 * s + j, a.q_bf16));
                most = fmaxf(most, m < __builtin_inff() ? m : __builtin_inff());
            }
        most = max32(most);
        // to [2^13, 2^14), by a power of two (2^100 at most)
        const int e = max((int)(__builtin_bit_cast(uint32_t, most) >> 23) - 127 - 13, -100);
        const float up = __builtin_bit_cast(float, (uint32_t)(127 - e) << 23);
        qk[n] = most < __builtin_inff() ? __builtin_bit_cast(float, (uint32_t)(127 + e) << 23) * a.scale : __builtin_nanf("");
        for (int s = 0; s < D / 16; s++)
            for (int j = 0; j < 8; j++) {
                const float x = value_at(a.q, at + 16 * s + j, a.q_bf16) * up;
                q[n][0][s][j] = (_Float16)x;
                if constexpr (P == 2) q[n][1][s][j] = (_Float16)(x - (float)q[n][0][s][j]);
            }
    }

    v16f o[NT][D / 32];
    float m_at[NT], base[NT], lim[NT], l_sum[NT];
#pragma unroll
    for (int n = 0; n < NT; n++) {
        m_at[n] = -__builtin_inff();
        base[n] = l_sum[n] = 0.0f;
        lim[n] = -__builtin_inff();  // t (less m) that is too large
#pragma unroll
        for (int d = 0; d < D / 32; d++)
#pragma unroll
            for (int r = 0; r < 16; r++) o[n][d][r] = 0.0f;
    }

    const int32_t *table = a.step.table + (int64_t)a.step.seq[i] * a.step.sequence_pages;
    const int last_block = (len - 1) / kKvBlock, in_mask = (1 << a.l.block_shift) - 1;
    auto block_at = [&](int tile, int b, int *in) -> const uint8_t * {
        const int blk = min(tile * 4 + b, last_block);
        *in = (head << a.l.block_shift) + (blk & in_mask);
        return a.l.base + (int64_t)max(table[blk >> a.l.block_shift], 0) * a.l.page_bytes;
    };
    uint4 kraw[N], vraw[N];
    float2 sraw = make_float2(0.0f, 0.0f);
    auto fetch = [&](int tile) {
#pragma unroll
        for (int j = 0; j < N; j++) {
            const int c = tid + 256 * j;
            if (4 * D % 256 == 0 || c < 4 * D) {
                int in;
                const int token = c / (D / 16);
                const uint8_t *pg = block_at(tile, token / kKvBlock, &in);
                kraw[j] = *(const uint4 *)(pg + in * (2 * kKvBlock * D) + token % kKvBlock * D + c % (D / 16) * 16);
                pg = block_at(tile, c / D, &in);
                vraw[j] = *(const uint4 *)(pg + in * (2 * kKvBlock * D) + kKvBlock * D + c % D * 16);
            }
        }
        if (tid < 4) {
            int in;
            const uint8_t *pg = block_at(tile, tid, &in);
            sraw = *(const float2 *)(pg + a.l.scales + 8 * in);
            if (tile * 4 + tid > last_block) sraw = make_float2(0.0f, 1.0f);
        }
    };
    auto stage = [&](int buf) {
#pragma unroll
        for (int j = 0; j < N; j++) {
            const int c = tid + 256 * j;
            if (4 * D % 256 == 0 || c < 4 * D) {
                uint32_t h[8];
                codes_to_half(kraw[j].x, h), codes_to_half(kraw[j].y, h + 2), codes_to_half(kraw[j].z, h + 4), codes_to_half(kraw[j].w, h + 6);
                uint4 *to = (uint4 *)&ks[buf][c / (D / 16)][c % (D / 16) * 16];
                to[0] = make_uint4(h[0], h[1], h[2], h[3]);
                to[1] = make_uint4(h[4], h[5], h[6], h[7]);
                codes_to_half(vraw[j].x, h), codes_to_half(vraw[j].z, h + 2), codes_to_half(vraw[j].y, h + 4), codes_to_half(vraw[j].w, h + 6);
                to = (uint4 *)&vs[buf][c % D][c / D * 16];
                to[0] = make_uint4(h[0], h[1], h[2], h[3]);
                to[1] = make_uint4(h[4], h[5], h[6], h[7]);
            }
        }
        if (tid < 4) {
            const float sv = sraw.y != sraw.y ? sraw.y : fmaxf(sraw.y, kKvMinScale);
            scales[buf][0][tid] = sraw.x;
            scales[buf][1][tid] = __builtin_amdgcn_logf(sv);
            scales[buf][2][tid] = sv == sv ? 1.0f / sv : 1.0f;
        }
    };

    if (t0 < t1) {
        fetch(vis.tile(t0));
        stage(0);
    }
    __syncthreads();
    for (int u = t0; u < t1; u++) {
        const int buf = (u - t0) & 1, tile = vis.tile(u), j0 = tile * kKvTile;
        if (u + 1 < t1) fetch(vis.tile(u + 1));
        // nothing of the tile that a row of the wave sees
        const bool hidden = j0 > p_last || (j0 + kKvTile - 1 <= p_first - a.window && j0 >= a.sinks) || w0 > r1;
        if (!hidden) {
            float sk[4], lv[4], rsv[4];
#pragma unroll
            for (int b = 0; b < 4; b++) sk[b] = scales[buf][0][b], lv[b] = scales[buf][1][b], rsv[b] = scales[buf][2][b];
            const bool whole = j0 + kKvTile - 1 <= p_first && (j0 > p_last - a.window || j0 + kKvTile - 1 < a.sinks);
#pragma unroll
            for (int sub = 0; sub < 2; sub++) {
                v16f s[NT];
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int r = 0; r < 16; r++) s[n][r] = 0.0f;
#pragma unroll
                for (int st = 0; st < D / 16; st++) {
                    const v8h k = *(const v8h *)&ks[buf][32 * sub + col][16 * st + 8 * half];
#pragma unroll
                    for (int n = 0; n < NT; n++)
#pragma unroll
                        for (int p = 0; p < P; p++) s[n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, q[n][p][st], s[n], 0, 0, 0);
                }
                v8h w[NT][P][2];
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    float t[16], top = -__builtin_inff();
#pragma unroll
                    for (int r = 0; r < 16; r++) t[r] = __builtin_fmaf(s[n][r], qk[n] * sk[2 * sub + r / 8], lv[2 * sub + r / 8] + base[n]);
                    if (!whole) {
#pragma unroll
                        for (int r = 0; r < 16; r++) {
                            const int at = j0 + 32 * sub + 8 * (r / 4) + 4 * half + r % 4;
                            if (!(at <= place[n] && (at > place[n] - a.window || at < a.sinks))) t[r] = -__builtin_inff();
                        }
                    }
#pragma unroll
                    for (int r = 0; r < 16; r++) top = fmaxf(top, t[r]);
                    if (__any(top > lim[n])) {
                        top = max32(top);
                        if (top > lim[n]) {  // m moves up to the largest t: by `up` octaves
                            const float up = top - (m_at[n] > -__builtin_inff() ? kUnit : 0.0f), f = m_at[n] > -__builtin_inff() ? __builtin_amdgcn_exp2f(-up) : 0.0f;
                            m_at[n] = m_at[n] > -__builtin_inff() ? m_at[n] + up : up;
                            const float shift = kUnit - m_at[n] - base[n];
                            base[n] = kUnit - m_at[n];
                            lim[n] = kUnit + kHead;
                            l_sum[n] *= f;
#pragma unroll
                            for (int r = 0; r < 16; r++) t[r] += shift;
#pragma unroll
                            for (int d = 0; d < D / 32; d++)
#pragma unroll
                                for (int r = 0; r < 16; r++) o[n][d][r] *= f;
                        }
                    }
#pragma unroll
                    for (int r = 0; r < 16; r++) {
                        const float e = __builtin_amdgcn_exp2f(t[r]);
                        l_sum[n] = __builtin_fmaf(e, rsv[2 * sub + r / 8], l_sum[n]);
                        w[n][0][r / 8][r % 8] = (_Float16)e;
                        if constexpr (P == 2) w[n][1][r / 8][r % 8] = (_Float16)(e - (float)w[n][0][r / 8][r % 8]);
                    }
                }
#pragma unroll
                for (int d = 0; d < D / 32; d++)
#pragma unroll
                    for (int k = 0; k < 2; k++) {
                        const v8h v = *(const v8h *)&vs[buf][32 * d + col][16 * (2 * sub + k) + 8 * half];
#pragma unroll
                        for (int n = 0; n < NT; n++)
#pragma unroll
                            for (int p = 0; p < P; p++) o[n][d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, w[n][p][k], o[n][d], 0, 0, 0);
                    }
            }
        }
        if (u + 1 < t1) stage(buf ^ 1);
        __syncthreads();
    }

#pragma unroll
    for (int n = 0; n < NT; n++) {
        const int r = w0 + n * 32 + col;
        const Two both = swap32(l_sum[n]);
        const float total = both.a + both.b;
        if (r > r1) continue;
        if (a.splits > 1) {
            const int64_t slot = (((int64_t)i * a.l.kv_heads + head) * a.max_rows + r) * a.splits + split;
#pragma unroll
            for (int d = 0; d < D / 32; d++)
#pragma unroll
                for (int g = 0; g < 4; g++)
                    *(float4 *)(a.part + slot * D + 32 * d + 8 * g + 4 * half) = make_float4(o[n][d][4 * g], o[n][d][4 * g + 1], o[n][d][4 * g + 2], o[n][d][4 * g + 3]);
            if (half == 0) {
                a.part_ml[2 * slot] = m_at[n];
                a.part_ml[2 * slot + 1] = total;
            }
        } else {
            const float f = total == 0.0f ? 0.0f : 1.0f / total;
            const int64_t to = (int64_t)(row0 + r / a.group) * a.out_stride + (head * a.group + r % a.group) * D + 4 * half;
#pragma unroll
            for (int d = 0; d < D / 32; d++)
#pragma unroll
                for (int g = 0; g < 4; g++) {
                    float4 x = make_float4(o[n][d][4 * g] * f, o[n][d][4 * g + 1] * f, o[n][d][4 * g + 2] * f, o[n][d][4 * g + 3] * f);
                    const int64_t at = to + 32 * d + 8 * g;
                    if (a.out_bf16) *(uint2 *)((uint16_t *)a.out + at) = make_uint2(bf16_bits(x.x) | bf16_bits(x.y) << 16, bf16_bits(x.z) | bf16_bits(x.w) << 16);
                    else *(float4 *)((float *)a.out + at) = x;
                }
        }
    }
}

template <int NT, int P>
hipError_t prefill(const KvAttend &a, hipStream_t s, hipEvent_t done) {
    const dim3 grid((unsigned)(a.l.kv_heads * a.splits), (unsigned)((a.max_rows + 128 * NT - 1) / (128 * NT)), (unsigned)a.step.n);
    switch (a.l.dim) {
    case 64: return launch_with_event(prefill_kernel<64, NT, P>, grid, dim3(256), s, done, a);
    case 96: return launch_with_event(prefill_kernel<96, NT, P>, grid, dim3(256), s, done, a);
    case 128: return launch_with_event(prefill_kernel<128, NT, P>, grid, dim3(256), s, done, a);
    case 192: return launch_with_event(prefill_kernel<192, NT, P>, grid, dim3(256), s, done, a);
    case 256: return launch_with_event(prefill_kernel<256, NT, P>, grid, dim3(256), s, done, a);
    }
    return hipErrorInvalidValue;
}

}  // namespace

hipError_t launch_kv_prefill(const KvAttend &a, hipStream_t s, hipEvent_t done) {
    hipEvent_t last = a.splits > 1 ? nullptr : done;
    const hipError_t e = a.out_bf16 ? prefill<1, 1>(a, s, last) : prefill<1, 2>(a, s, last);
    return e == hipSuccess && a.splits > 1 ? launch_kv_join(a, s, done) : e;
}

}  // namespace j4q
