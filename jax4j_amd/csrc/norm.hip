// Norms before and after a block of a decoder, with the block's gate and the residual between them (j4q_norm_into):
//   h = residual + scale gate after(block),  out = before(h),
// each norm x / sqrt(mean(x^2) + eps) w + b, or of x - mean(x). Engine-local; the reference has no norms on this path.
//
// Bound by memory: a row is read once, kept in registers (beyond 16384 values in LDS) from the first sum to the last product, and written
// once. A team of 64, 256 or 1024 threads has a row, 8 values a thread and pass: 16 bytes of bf16, or twice 16 of fp32, where addresses and
// strides allow, else value after value across the team. Sums of values and squares are in 64 bits: they neither overflow nor lose
// what a mean far from 0 hides, and cost nothing beside the memory. 16381 rows of 4096, a norm on either side of the residual and a gate:
// 162 us, 5.0 TB/s. Few rows wait for their sums, so these take no LDS within a wave and no division (1021 rows of 1152, two norms with
// means: 8.8 us with them, 7.7 without; all loads of a row ahead of its first sum: no faster).
#include "arguments.h"
#include "engine.h"
#include "teams.h"

namespace j4q {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

struct NormK {
    int kind;  // 0: none
    float eps, add;
    const float *weight, *bias;
};
struct NormP {
    const uint8_t *residual, *block, *gate;
    uint8_t *residual_out, *out;
    int64_t rows;
    uint32_t gate_every;
    int64_t residual_stride, block_stride, gate_stride, residual_out_stride, out_stride;  // bytes
    int dim;
    double inv_dim;
    bool residual16, block16, gate16, out16;  // bf16
    float scale;
    NormK after, before;
};

// (by value: a bit cast of a vector's element itself takes the first one)
__device__ __forceinline__ float as_float(uint32_t b) { return __builtin_bit_cast(float, b); }

// The 8 values of a thread and pass as they lie in memory.
struct Raw {
    u32x4 v[2];
};

// VEC: thread t has values 8 (t + T c) .. + 7 in pass c; else t + T (8 c + j).
template <int T, bool VEC>
struct At {
    static __device__ __forceinline__ int of(int t, int c, int j) { return VEC ? 8 * (t + T * c) + j : t + T * (8 * c + j); }
};

template <int T, bool VEC>
__device__ __forceinline__ void load(Raw &r, const uint8_t *row, bool half, int t, int c, int dim) {
    if constexpr (VEC) {
        const int i = At<T, true>::of(t, c, 0);
        if (i < dim) {
            if (half) {
                r.v[0] = *reinterpret_cast<const u32x4 *>(row + 2 * (int64_t)i);
            } else {
                r.v[0] = *reinterpret_cast<const u32x4 *>(row + 4 * (int64_t)i);
                r.v[1] = *reinterpret_cast<const u32x4 *>(row + 4 * (int64_t)i + 16);
            }
        } else {
            r.v[0] = r.v[1] = u32x4{};
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int i = At<T, false>::of(t, c, j);
            uint32_t v = 0;
            if (i < dim) v = half ? (uint32_t)reinterpret_cast<const uint16_t *>(row)[i] << 16 : reinterpret_cast<const uint32_t *>(row)[i];
            r.v[j >> 2][j & 3] = v;
        }
    }
}

template <bool VEC>
__device__ __forceinline__ f32x8 values(const Raw &r, bool half) {
    f32x8 x;
    if (VEC && half) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            x[2 * j] = as_float(r.v[0][j] << 16);
            x[2 * j + 1] = as_float(r.v[0][j] & 0xFFFF0000u);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = as_float(r.v[j >> 2][j & 3]);
    }
    return x;
}

// Rounded to bf16 once, to nearest even.
__device__ __forceinline__ uint32_t pair_bf16(float a, float b) { return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), bf16x2)); }

template <int T, bool VEC>
__device__ __forceinline__ void store(const f32x8 &x, uint8_t *row, bool half, int t, int c, int dim) {
    if constexpr (VEC) {
        const int i = At<T, true>::of(t, c, 0);
        if (i >= dim) return;
        if (half) {
            *reinterpret_cast<u32x4 *>(row + 2 * (int64_t)i) = u32x4{pair_bf16(x[0], x[1]), pair_bf16(x[2], x[3]), pair_bf16(x[4], x[5]), pair_bf16(x[6], x[7])};
        } else {
            typedef float f32x4 __attribute__((ext_vector_type(4)));
            *reinterpret_cast<f32x4 *>(row + 4 * (int64_t)i) = f32x4{x[0], x[1], x[2], x[3]};
            *reinterpret_cast<f32x4 *>(row + 4 * (int64_t)i + 16) = f32x4{x[4], x[5], x[6], x[7]};
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int i = At<T, false>::of(t, c, j);
            if (i >= dim) continue;
            if (half) reinterpret_cast<uint16_t *>(row)[i] = (uint16_t)pair_bf16(x[j], x[j]);
            else reinterpret_cast<float *>(row)[i] = x[j];
        }
    }
}

// 1 / sqrt(v): v_rsq_f64, good to some 24 bits, and a step of Newton's.
__device__ __forceinline__ double inverse_root(double v) {
    const double y = __builtin_amdgcn_rsq(v), e = fma(-v * y, y, 1.0);
    return e == e ? fma(0.5 * y, e, y) : y;  // not of 0 or infinity
}

// A root's inverse y beyond 32 bits, or with fewer of them, and the power of two that the values take of it first. The same in a whole team.
__device__ __forceinline__ bool far(double y) { return y > 0x1p126 || y < 0x1p-126; }
__device__ __forceinline__ int far_power(double y) { return y > 1. ? 100 : -64; }

// Sum over the team's T threads, in the same order whichever row of the workgroup the team has. `slot`: T / 64 doubles of the team.
template <int T>
__device__ __forceinline__ double row_sum(double v, double *slot, int t) {
    v = team_sum<64>(v);
    if constexpr (T > 64) {
        __syncthreads();  // the sum before has been read
        if ((t & 63) == 0) slot[t >> 6] = v;
        __syncthreads();
        v = slot[0];
#pragma unroll
        for (int w = 1; w < T / 64; w++) v += slot[w];
    }
    return v;
}

// The quotient itself where it is exact: rows of equal values have no rest.
__device__ __forceinline__ double mean_of(double sum, int dim, double inv_dim) {
    const double near = sum * inv_dim;
    return fma(fma(-near, (double)dim, sum), inv_dim, near);
}

template <int T, int C, bool VEC>
__device__ __forceinline__ void apply(const NormK &k, f32x8 (&x)[C], Raw (&w)[C], Raw (&b)[C], double *slot, int t, int dim, double inv_dim) {
    double mean = 0;
    if (k.kind == J4Q_NORM_LAYER) {
#pragma unroll
        for (int c = 0; c < C; c++)
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (At<T, VEC>::of(t, c, j) < dim) mean += (double)x[c][j];
        mean = mean_of(row_sum<T>(mean, slot, t), dim, inv_dim);
    }
    double sum = 0;
#pragma unroll
    for (int c = 0; c < C; c++)
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (At<T, VEC>::of(t, c, j) < dim) {
                const double d = (double)x[c][j] - mean;
                sum = fma(d, d, sum);
                x[c][j] = (float)d;
            }
    double root = inverse_root(fma(row_sum<T>(sum, slot, t), inv_dim, (double)k.eps));
    if (far(root)) {
        const int power = far_power(root);
        root = ldexp(root, -power);
#pragma unroll
        for (int c = 0; c < C; c++) x[c] *= ldexpf(1.f, power);
    }
    const float inv = (float)root;
#pragma unroll
    for (int c = 0; c < C; c++) {
        if (k.weight) load<T, VEC>(w[c], (const uint8_t *)k.weight, false, t, c, dim);
        if (k.bias) load<T, VEC>(b[c], (const uint8_t *)k.bias, false, t, c, dim);
    }
#pragma unroll
    for (int c = 0; c < C; c++)
#pragma unroll
        for (int j = 0; j < 8; j++) {
            float v = x[c][j] * inv;
            if (k.weight) v *= as_float(w[c].v[j >> 2][j & 3]) + k.add;
            if (k.bias) v += as_float(b[c].v[j >> 2][j & 3]);
            x[c][j] = v;
        }
}

// G teams of T threads a workgroup, a row each; C passes of 8 T values.
template <int T, int C, bool VEC>
__global__ void __launch_bounds__(T < 256 ? 256 : T)
norm_kernel(NormP p) {
    constexpr int G = T < 256 ? 256 / T : 1;
    __shared__ double slots[T / 64];
    const int t = (int)threadIdx.x % T;
    const int64_t row = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * G + threadIdx.x / T;
    if (row >= p.rows) return;  // teams of more than a wave have a workgroup each: whole workgroups leave
    const uint8_t *const g = p.gate + (p.gate_every ? (uint32_t)row / p.gate_every : 0) * p.gate_stride;
    // Registers of each part's own, which the compiler then loads a pass ahead (16381 rows of 4096: 165 -> 162 us).
    Raw res[C], blk[C], gate[C], w[2][C], b[2][C];
    if (p.block) {
#pragma unroll
        for (int c = 0; c < C; c++) load<T, VEC>(blk[c], p.block + row * p.block_stride, p.block16, t, c, p.dim);
    }
    if (p.residual) {
#pragma unroll
        for (int c = 0; c < C; c++) load<T, VEC>(res[c], p.residual + row * p.residual_stride, p.residual16, t, c, p.dim);
    }
    f32x8 x[C];
    if (p.block) {
#pragma unroll
        for (int c = 0; c < C; c++) x[c] = values<VEC>(blk[c], p.block16);
        if (p.after.kind) apply<T, C, VEC>(p.after, x, w[0], b[0], slots, t, p.dim, p.inv_dim);
        if (p.gate) {
#pragma unroll
            for (int c = 0; c < C; c++) {
                load<T, VEC>(gate[c], g, p.gate16, t, c, p.dim);
                x[c] *= values<VEC>(gate[c], p.gate16);
            }
        }
#pragma unroll
        for (int c = 0; c < C; c++) x[c] *= p.scale;
    } else {
#pragma unroll
        for (int c = 0; c < C; c++) x[c] = f32x8{};
    }
    if (p.residual) {
#pragma unroll
        for (int c = 0; c < C; c++) x[c] += values<VEC>(res[c], p.residual16);
    }
    if (p.residual_out) {
#pragma unroll
        for (int c = 0; c < C; c++) store<T, VEC>(x[c], p.residual_out + row * p.residual_out_stride, p.residual16, t, c, p.dim);
    }
    if (!p.before.kind) return;
    apply<T, C, VEC>(p.before, x, w[1], b[1], slots, t, p.dim, p.inv_dim);
#pragma unroll
    for (int c = 0; c < C; c++) store<T, VEC>(x[c], p.out + row * p.out_stride, p.out16, t, c, p.dim);
}

// Rows beyond 16384, 32 values of 1024 threads: they lie in LDS, of which each thread has its own, and go through registers 8 at a time. (In
// registers, 128 a thread, they spilled 142 of them: 2000 rows of 20000, two norms and the residual, 470 us; here 115, 2.8 TB/s, and of
// 20001, value by value, 203.) The sums' order is that of norm_kernel.
template <bool VEC>
__global__ void __launch_bounds__(1024)
norm_long_kernel(NormP p) {
    constexpr int T = 1024, C = 4;
    __shared__ float held[C * 8 * T];
    __shared__ double slots[T / 64];
    const int t = (int)threadIdx.x, dim = p.dim, passes = (dim + 8 * T - 1) / (8 * T);
    const int64_t row = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
    if (row >= p.rows) return;
    const uint8_t *const g = p.gate + (p.gate_every ? (uint32_t)row / p.gate_every : 0) * p.gate_stride;
    auto put = [&](int c, const f32x8 &x) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < 8; j++) held[(8 * c + j) * T + t] = x[j];
    };
    auto get = [&](int c) __attribute__((always_inline)) {
        f32x8 x;
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = held[(8 * c + j) * T + t];
        return x;
    };
    auto read = [&](const uint8_t *at, bool half, int c) __attribute__((always_inline)) {
        Raw r;
        load<T, VEC>(r, at, half, t, c, dim);
        return values<VEC>(r, half);
    };
    auto apply = [&](const NormK &k) __attribute__((always_inline)) {
        double mean = 0;
        if (k.kind == J4Q_NORM_LAYER) {
#pragma unroll 1
            for (int c = 0; c < passes; c++) {
                const f32x8 x = get(c);
#pragma unroll
                for (int j = 0; j < 8; j++)
                    if (At<T, VEC>::of(t, c, j) < dim) mean += (double)x[j];
            }
            mean = mean_of(row_sum<T>(mean, slots, t), dim, p.inv_dim);
        }
        double sum = 0;
#pragma unroll 1
        for (int c = 0; c < passes; c++) {
            f32x8 x = get(c);
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (At<T, VEC>::of(t, c, j) < dim) {
                    const double d = (double)x[j] - mean;
                    sum = fma(d, d, sum);
                    x[j] = (float)d;
                }
            if (k.kind == J4Q_NORM_LAYER) put(c, x);
        }
        const double root = inverse_root(fma(row_sum<T>(sum, slots, t), p.inv_dim, (double)k.eps));
        const int power = far(root) ? far_power(root) : 0;
        const float first = ldexpf(1.f, power), inv = (float)ldexp(root, -power);
#pragma unroll 1
        for (int c = 0; c < passes; c++) {
            f32x8 x = get(c);
            x *= first;
            x *= inv;
            if (k.weight) x *= read((const uint8_t *)k.weight, false, c) + k.add;
            if (k.bias) x += read((const uint8_t *)k.bias, false, c);
            put(c, x);
        }
    };
    if (p.block) {
#pragma unroll 1
        for (int c = 0; c < passes; c++) put(c, read(p.block + row * p.block_stride, p.block16, c));
        if (p.after.kind) apply(p.after);
    }
#pragma unroll 1
    for (int c = 0; c < passes; c++) {
        f32x8 x = {};
        if (p.block) {
            x = get(c);
            if (p.gate) x *= read(g, p.gate16, c);
            x *= p.scale;
        }
        if (p.residual) x += read(p.residual + row * p.residual_stride, p.residual16, c);
        if (p.residual_out) store<T, VEC>(x, p.residual_out + row * p.residual_out_stride, p.residual16, t, c, dim);
        put(c, x);
    }
    if (!p.before.kind) return;
    apply(p.before);
#pragma unroll 1
    for (int c = 0; c < passes; c++) store<T, VEC>(get(c), p.out + row * p.out_stride, p.out16, t, c, dim);
}

template <int G>
dim3 grid_of(const NormP &p) {
    const int64_t groups = (p.rows + G - 1) / G, x = groups < 1 << 20 ? groups : 1 << 20;  // a grid's threads are counted in 32 bits
    return dim3((unsigned)x, (unsigned)((groups + x - 1) / x));
}

template <int T, int C>
hipError_t launch(const NormP &p, bool vec, hipStream_t s) {
    constexpr int G = T < 256 ? 256 / T : 1;
    if (vec) norm_kernel<T, C, true><<<grid_of<G>(p), T * G, 0, s>>>(p);
    else norm_kernel<T, C, false><<<grid_of<G>(p), T * G, 0, s>>>(p);
    return hipGetLastError();
}

hipError_t launch_norm(const NormP &p, bool vec, hipStream_t s) {
    if (p.dim <= 512) return launch<64, 1>(p, vec, s);
    if (p.dim <= 1024) return launch<64, 2>(p, vec, s);
    if (p.dim <= 2048) return launch<256, 1>(p, vec, s);
    if (p.dim <= 4096) return launch<256, 2>(p, vec, s);
    if (p.dim <= 8192) return launch<256, 4>(p, vec, s);
    if (p.dim <= 16384) return launch<1024, 2>(p, vec, s);
    if (vec) norm_long_kernel<true><<<grid_of<1>(p), 1024, 0, s>>>(p);
    else norm_long_kernel<false><<<grid_of<1>(p), 1024, 0, s>>>(p);
    return hipGetLastError();
}

int check_norm(const char *which, const j4q_norm *n, NormK *out) {
    *out = NormK{};
    if (!n) return J4Q_OK;
    if (n->kind != J4Q_NORM_RMS && n->kind != J4Q_NORM_LAYER)
        return report_error(J4Q_EUNSUPPORTED, "norm_into: kind %d of the norm %s (J4Q_NORM_RMS or J4Q_NORM_LAYER)", n->kind, which);
    if (!(n->eps >= 0.f)) return report_error(J4Q_EINVAL, "norm_into: eps of the norm %s must not be negative", which);
    if (!aligned(n->weight, 4) || !aligned(n->bias, 4)) return report_error(J4Q_EINVAL, "norm_into: weight and bias of the norm %s must be 4-byte aligned", which);
    *out = NormK{n->kind, n->eps, n->weight_add, n->weight, n->bias};
    return J4Q_OK;
}

}  // namespace
}  // namespace j4q

using namespace j4q;

extern "C" int j4q_norm_into(const j4q_norm_args *a, void *stream) {
    if (!a) return report_error(J4Q_EINVAL, "norm_into: NULL argument");
    if (!a->residual && !a->block) return report_error(J4Q_EINVAL, "norm_into: neither a residual nor a block");
    if (!a->residual_out && !a->out) return report_error(J4Q_EINVAL, "norm_into: neither residual_out nor out");
    if (!a->out != !a->before) return report_error(J4Q_EINVAL, "norm_into: out and the norm before the next block go together");
    if (!a->block && (a->gate || a->after)) return report_error(J4Q_EINVAL, "norm_into: a gate or a norm behind a block that is not there");
    if (!dense_type(a->residual_type) || !dense_type(a->block_type) || !dense_type(a->gate_type) || !dense_type(a->out_type))
        return report_error(J4Q_EUNSUPPORTED, "norm_into: types %d, %d, %d, %d (J4Q_KIND_F32 or J4Q_KIND_BF16)", a->residual_type, a->block_type, a->gate_type, a->out_type);
    if (a->rows < 1 || a->rows > 1 << 30 || a->dim < 1) return report_error(J4Q_EINVAL, "norm_into: %lld rows of %d values", (long long)a->rows, a->dim);
    if (a->dim > 32768) return report_error(J4Q_EUNSUPPORTED, "norm_into: rows of %d values (at most 32768)", a->dim);
    if (a->gate_every < 0) return report_error(J4Q_EINVAL, "norm_into: %lld rows to a gate", (long long)a->gate_every);
    NormP p{};
    int rc;
    if ((rc = check_norm("behind the block", a->after, &p.after)) || (rc = check_norm("before the next block", a->before, &p.before))) return rc;
    struct Part {
        const void *p;
        int64_t stride, rows;
        int type;
        bool written;
    };
    const int64_t gates = a->gate_every ? (a->rows - 1) / a->gate_every + 1 : 1;
    const Part part[5] = {{a->residual, a->residual_stride, a->rows, a->residual_type, false},
                          {a->block, a->block_stride, a->rows, a->block_type, false},
                          {a->gate, a->gate_stride, gates, a->gate_type, false},
                          {a->residual_out, a->residual_out_stride, a->rows, a->residual_type, true},
                          {a->out, a->out_stride, a->rows, a->out_type, true}};
    int64_t stride[5];
    bool vec = a->dim % 8 == 0;
    for (const NormK *k : {&p.after, &p.before}) vec &= aligned(k->weight, 16) && aligned(k->bias, 16);
    for (int i = 0; i < 5; i++) {
        const int64_t e = dense_size(part[i].type);
        stride[i] = part[i].stride ? part[i].stride : a->dim;
        if (!part[i].p) continue;
        if (stride[i] < a->dim || stride[i] > 1ll << 40 || stride[i] > (INT64_MAX >> 3) / part[i].rows)
            return report_error(J4Q_EINVAL, "norm_into: rows of %d values %lld apart", a->dim, (long long)stride[i]);
        stride[i] *= e;
        if (!aligned(part[i].p, (uintptr_t)e)) return report_error(J4Q_EINVAL, "norm_into: pointers must be aligned to their values");
        vec &= aligned(part[i].p, 16) && stride[i] % 16 == 0;
    }
    const int64_t dim = a->dim;
    for (int i = 3; i < 5; i++) {  // an output and anything else: the very same rows of a thread's values, or apart
        if (!part[i].p) continue;
        const int64_t e = dense_size(part[i].type);
        for (int j = 0; j < i; j++) {
            if (!part[j].p) continue;
            const int64_t f = dense_size(part[j].type);
            const bool same = part[i].p == part[j].p && stride[i] == stride[j] && e == f && j < 2;
            const bool apart = part[j].rows == part[i].rows ? !overlap(part[i].p, stride[i], dim * e, part[j].p, stride[j], dim * f, a->rows)
                                                            : !overlap(part[i].p, (uint64_t)((part[i].rows - 1) * stride[i] + dim * e), part[j].p,
                                                                       (uint64_t)((part[j].rows - 1) * stride[j] + dim * f));
            if (!same && !apart) return report_error(J4Q_EUNSUPPORTED, "norm_into: an output overlaps an input or the other output without being that input itself");
        }
        for (const NormK *k : {&p.after, &p.before})
            for (const float *w : {k->weight, k->bias})
                if (w && overlap(part[i].p, (uint64_t)((part[i].rows - 1) * stride[i] + dim * e), w, (uint64_t)dim * 4))
                    return report_error(J4Q_EUNSUPPORTED, "norm_into: an output overlaps a norm's weights");
    }
    p.residual = (const uint8_t *)a->residual;
    p.block = (const uint8_t *)a->block;
    p.gate = (const uint8_t *)a->gate;
    p.residual_out = (uint8_t *)a->residual_out;
    p.out = (uint8_t *)a->out;
    p.rows = a->rows;
    p.inv_dim = 1.0 / (double)a->dim;
    p.gate_every = (uint32_t)(a->gate_every < a->rows ? a->gate_every : a->rows);
    p.residual_stride = stride[0];
    p.block_stride = stride[1];
    p.gate_stride = stride[2];
    p.residual_out_stride = stride[3];
    p.out_stride = stride[4];
    p.dim = a->dim;
    p.residual16 = a->residual_type == J4Q_KIND_BF16;
    p.block16 = a->block_type == J4Q_KIND_BF16;
    p.gate16 = a->gate_type == J4Q_KIND_BF16;
    p.out16 = a->out_type == J4Q_KIND_BF16;
    p.scale = a->scale;
    std::lock_guard<std::mutex> lk(abi::lock());
    if ((rc = abi::ready_locked())) return rc;
    const hipError_t e = launch_norm(p, vec, stream ? (hipStream_t)stream : abi::stream());
    return e == hipSuccess ? J4Q_OK : report_hip("norm_into", e);
}
