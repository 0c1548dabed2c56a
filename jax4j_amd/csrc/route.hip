// Routing of tokens to experts (j4q_route_into): the top_k experts of every row of logits and their weights. Engine-local; the
// reference has no experts.
//
// What a row needs is small (a read of its logits); what it costs is the choice, so a team of 16 lanes has a row of up to 128
// experts (four rows a wave) and of 64 lanes the others, each lane J experts l + L j in registers. Keys are whole numbers in the order
// of the values they stand for, 0 where nothing may be chosen: without bias and groups the logits' own 32 bits, else 64 bits of score
// + bias (or the logit), where rounding cannot exchange two sums that 32 bits would not tell apart. A choice is the maximum of the keys'
// 32 bits (of 64: of the upper ones, then of the lower ones where the upper are that) and the lowest index that has it, each over the
// lane's own and then over the team. Instructions bound it, and
// where rows are few the chain of maxima: 8 of 128 experts, 16381 rows 7.8 us (9.8 with keys of 64 bits and exchanges through LDS), 8 of 256 in groups, 61
// rows 9.5 (12.7).
// Lane s of the team then has slot s, reads that expert's logit once more and computes its weight.
#include "arguments.h"
#include "engine.h"
#include "teams.h"

namespace j4q {
namespace {

constexpr float kInf = __builtin_inff();

struct RouteP {
    const uint8_t *logits;
    const float *bias;
    int32_t *ids;
    float *weights;
    int64_t rows, stride;  // bytes
    int experts, top, groups, top_groups, best;
    bool half, sigmoid, renormalize;
    float scale;
};

// Whole numbers in the order of the numbers, all above 0 (NaN apart).
__device__ __forceinline__ uint32_t order32(float v) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v == 0.f ? 0.f : v);  // -0 is 0
    return u >> 31 ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ uint64_t order64(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v == 0. ? 0. : v);
    return u >> 63 ? ~u : u | 0x8000000000000000ull;
}
__device__ __forceinline__ double unorder64(uint64_t k) { return __builtin_bit_cast(double, k >> 63 ? k & 0x7fffffffffffffffull : ~k); }

__device__ __forceinline__ float logit_of(const RouteP &p, int64_t row, int i) {
    const uint8_t *const at = p.logits + row * p.stride;
    const float v = p.half ? __builtin_bit_cast(float, (uint32_t)reinterpret_cast<const uint16_t *>(at)[i] << 16) : reinterpret_cast<const float *>(at)[i];
    return v == v ? v : -kInf;
}

// WIDE: keys of 64 bits (a bias, or groups). 256 / L rows a workgroup.
template <int L, int J, bool WIDE>
__global__ void __launch_bounds__(256)
route_kernel(RouteP p) {
    constexpr int R = 256 / L;
    __shared__ uint64_t keys[WIDE ? R : 1][WIDE ? L * J : 1];
    const int t = (int)threadIdx.x % L, team = (int)threadIdx.x / L;
    const int64_t row = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * R + team;
    if (row >= p.rows) return;  // whole teams, which meet nowhere but in their own wave
    float x[J], top = -kInf;
#pragma unroll
    for (int j = 0; j < J; j++) {
        x[j] = t + L * j < p.experts ? logit_of(p, row, t + L * j) : -kInf;
        top = fmaxf(top, x[j]);
    }
    float sum = 0.f;
    if (!p.sigmoid) {
        top = team_max<L>(top);
#pragma unroll
        for (int j = 0; j < J; j++) sum += x[j] == -kInf ? 0.f : x[j] == top ? 1.f : expf(x[j] - top);  // (inf - inf is no number)
        sum = team_sum<L>(sum);
    }
    // Groups' two best are summed as scores, bias or not: sums of logits are not in the order of sums of scores, and a constant added
    // to a row, which changes no softmax, moves a group's two logits twice as far as the one of a group that has no more.
    const bool scored = WIDE && (p.bias || (p.groups > 1 && p.best == 2));
    uint64_t key[J];
#pragma unroll
    for (int j = 0; j < J; j++) {
        if constexpr (WIDE) {
            double c = x[j];
            if (scored && x[j] > -kInf) c = p.sigmoid ? 1. / (1. + exp(-(double)x[j])) : x[j] == top ? 1. : exp((double)x[j] - (double)top);
            key[j] = __builtin_bit_cast(uint64_t, c);
        } else {
            key[j] = x[j] > -kInf ? (uint64_t)order32(x[j]) << 32 : 0;
        }
    }
    if constexpr (WIDE) {
        double total = 1.;
        if (scored && !p.sigmoid) {  // the softmax in 64 bits
            total = 0.;
#pragma unroll
            for (int j = 0; j < J; j++) total += x[j] > -kInf ? __builtin_bit_cast(double, key[j]) : 0.;
            total = team_sum<L>(total);
        }
#pragma unroll
        for (int j = 0; j < J; j++) {
            const int i = t + L * j;
            double c = __builtin_bit_cast(double, key[j]);
            if (scored && x[j] > -kInf) c = c / total + (p.bias ? (double)p.bias[i] : 0.);
            key[j] = x[j] > -kInf && c > (double)-kInf ? order64(c) : 0;
        }
        if (p.groups > 1) {
            const int size = p.experts / p.groups;
#pragma unroll
            for (int j = 0; j < J; j++) keys[team][t + L * j] = key[j];
            asm volatile("" ::: "memory");  // the team is part of one wave, whose LDS operations are in order
            // lane g has group g: its rank, and how many groups come before it
            uint64_t one = 0, two = 0;
            if (t < p.groups)
                for (int i = 0; i < size; i++) {
                    const uint64_t k = keys[team][t * size + i];
                    two = k > one ? one : k > two ? k : two;
                    one = k > one ? k : one;
                }
            uint64_t rank = one;
            if (p.best == 2 && two) {
                const double r = unorder64(one) + unorder64(two);
                rank = r == r ? order64(r) : one;  // inf - inf
            }
            int before = 0;
            for (int g = 0; g < p.groups; g++) {
                const uint64_t other = __shfl(rank, g, L);
                before += other > rank || (other == rank && g < t);
            }
            const uint64_t open = __ballot(t < p.groups && before < p.top_groups) >> ((threadIdx.x & 63) / L * L);
#pragma unroll
            for (int j = 0; j < J; j++)
                if (!(open >> ((t + L * j) / size & 63) & 1)) key[j] = 0;  // (past the experts keys are 0)
            if (scored && !p.bias) {  // inside the open groups the logits decide, which tell apart what scores round to the same
#pragma unroll
                for (int j = 0; j < J; j++) key[j] = key[j] ? order64((double)x[j]) : 0;
            }
        }
    }
    // Slot s of the row goes to lane s.
    uint32_t upper[J], lower[WIDE ? J : 1];
#pragma unroll
    for (int j = 0; j < J; j++) {
        upper[j] = (uint32_t)(key[j] >> 32);
        if constexpr (WIDE) lower[j] = (uint32_t)key[j];
    }
    int mine = -1;
    for (int s = 0; s < p.top; s++) {
        uint32_t best = 0, low = 0;
#pragma unroll
        for (int j = 0; j < J; j++) best = upper[j] > best ? upper[j] : best;
        best = team_max<L>(best);
        if (best == 0) break;  // the same in the whole team; no key above 0 has upper bits of 0
        if constexpr (WIDE) {
#pragma unroll
            for (int j = 0; j < J; j++) low = upper[j] == best && lower[j] > low ? lower[j] : low;
            low = team_max<L>(low);
        }
        int at = L * J;
#pragma unroll
        for (int j = J - 1; j >= 0; j--) {
            bool is = upper[j] == best;
            if constexpr (WIDE) is = is && lower[j] == low;
            at = is ? t + L * j : at;
        }
        at = team_min<L>(at);
        if (t == s) mine = at;
#pragma unroll
        for (int j = 0; j < J; j++) upper[j] = t + L * j == at ? 0 : upper[j];
    }
    float w = 0.f, part = 0.f;
    const float own = mine >= 0 ? logit_of(p, row, mine) : -kInf;
    if (p.sigmoid) {
        // divided by their sum, scores may have a factor in common: e^-m, m the largest chosen logit where that is below 0, so
        // that scores too small for 32 bits still have their shares
        const float most = p.renormalize ? fminf(team_max<L>(own), 0.f) : 0.f;
        if (mine >= 0) w = own < 0.f ? expf(own - most) / (1.f + expf(own)) : 1.f / (1.f + expf(-own));
        part = w;
    } else {
        // likewise: what a bias or a group keeps out may lie so far above that beside it all chosen scores are 0
        const float most = p.renormalize ? team_max<L>(own) : top;
        if (mine >= 0) w = own == most ? 1.f : expf(own - most);
        part = w;
        if (!p.renormalize) w /= sum;
    }
    if (p.renormalize) {
        part = team_sum<L>(part);
        w = part > 0.f ? w / part : 0.f;
    }
    if (t < p.top) {
        p.ids[row * p.top + t] = mine;
        p.weights[row * p.top + t] = mine >= 0 ? w * p.scale : 0.f;
    }
}

template <int L, int J>
hipError_t launch(const RouteP &p, hipStream_t s) {
    const int64_t groups = (p.rows + 256 / L - 1) / (256 / L), x = groups < 1 << 20 ? groups : 1 << 20;
    const dim3 grid((unsigned)x, (unsigned)((groups + x - 1) / x));
    if (p.bias || p.groups > 1) route_kernel<L, J, true><<<grid, 256, 0, s>>>(p);
    else route_kernel<L, J, false><<<grid, 256, 0, s>>>(p);
    return hipGetLastError();
}

hipError_t launch_route(const RouteP &p, hipStream_t s) {
    if (p.top <= 16 && p.groups <= 16) {
        if (p.experts <= 32) return launch<16, 2>(p, s);
        if (p.experts <= 64) return launch<16, 4>(p, s);
        if (p.experts <= 128) return launch<16, 8>(p, s);
    }
    if (p.experts <= 128) return launch<64, 2>(p, s);
    if (p.experts <= 256) return launch<64, 4>(p, s);
    if (p.experts <= 512) return launch<64, 8>(p, s);
    return launch<64, 16>(p, s);
}

}  // namespace
}  // namespace j4q

using namespace j4q;

extern "C" int j4q_route_into(const j4q_route_args *a, void *stream) {
    if (!a || !a->logits || !a->ids || !a->weights) return report_error(J4Q_EINVAL, "route_into: NULL argument");
    if (!dense_type(a->type)) return report_error(J4Q_EUNSUPPORTED, "route_into: type %d (J4Q_KIND_F32 or J4Q_KIND_BF16)", a->type);
    if (a->score != J4Q_ROUTE_SOFTMAX && a->score != J4Q_ROUTE_SIGMOID) return report_error(J4Q_EUNSUPPORTED, "route_into: unknown score %d", a->score);
    if (a->rows < 1 || a->rows > 1 << 30 || a->experts < 1 || a->experts > 1024)
        return report_error(J4Q_EINVAL, "route_into: %lld rows of %d experts (1 to 1024)", (long long)a->rows, a->experts);
    const int groups = a->groups ? a->groups : 1, top_groups = groups > 1 ? a->top_groups : 1;
    if (groups < 1 || groups > 64 || a->experts % groups || top_groups < 1 || top_groups > groups)
        return report_error(J4Q_EINVAL, "route_into: %d of %d groups of %d experts (equal groups, at most 64)", top_groups, groups, a->experts);
    if (groups > 1 && a->group_best != 1 && a->group_best != 2) return report_error(J4Q_EINVAL, "route_into: groups by their %d best (1 or 2)", a->group_best);
    if (a->top_k < 1 || a->top_k > 64 || a->top_k > a->experts / groups * top_groups)
        return report_error(J4Q_EINVAL, "route_into: %d of %d experts (at most 64)", a->top_k, a->experts / groups * top_groups);
    const int64_t e = dense_size(a->type), stride = a->stride ? a->stride : a->experts;
    if (stride < a->experts || stride > 1ll << 30) return report_error(J4Q_EINVAL, "route_into: rows of %d logits %lld values apart", a->experts, (long long)stride);
    if (!aligned(a->logits, (uintptr_t)e) || !aligned(a->bias, 4) || !aligned(a->ids, 4) || !aligned(a->weights, 4))
        return report_error(J4Q_EINVAL, "route_into: pointers must be aligned to their values");
    const uint64_t in = (uint64_t)((a->rows - 1) * stride + a->experts) * (uint64_t)e, out = (uint64_t)a->rows * (uint64_t)a->top_k * 4;
    if (overlap(a->logits, in, a->ids, out) || overlap(a->logits, in, a->weights, out) || overlap(a->ids, out, a->weights, out) ||
        (a->bias && (overlap(a->bias, (uint64_t)a->experts * 4, a->ids, out) || overlap(a->bias, (uint64_t)a->experts * 4, a->weights, out))))
        return report_error(J4Q_EUNSUPPORTED, "route_into: ids and weights must lie apart from the inputs and each other");
    RouteP p{};
    p.logits = (const uint8_t *)a->logits;
    p.bias = a->bias;
    p.ids = a->ids;
    p.weights = a->weights;
    p.rows = a->rows;
    p.stride = stride * e;
    p.experts = a->experts;
    p.top = a->top_k;
    p.groups = groups;
    p.top_groups = top_groups;
    p.best = a->group_best;
    p.half = a->type == J4Q_KIND_BF16;
    p.sigmoid = a->score == J4Q_ROUTE_SIGMOID;
    p.renormalize = a->renormalize != 0;
    p.scale = a->scale;
    std::lock_guard<std::mutex> lk(abi::lock());
    int rc;
    if ((rc = abi::ready_locked())) return rc;
    const hipError_t err = launch_route(p, stream ? (hipStream_t)stream : abi::stream());
    return err == hipSuccess ? J4Q_OK : report_hip("route_into", err);
}
