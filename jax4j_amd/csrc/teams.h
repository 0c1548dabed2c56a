// Sums and maxima over teams of 16 or 64 lanes of a wave.
#pragma once

#include <stdint.h>

namespace j4q {
namespace {

// v of this lane and of its partner of step O = 1, 2, 4, ...: within 16 lanes by data-parallel primitives (the steps 4 and 8 mirror 8 or 16
// lanes, which hold one value in each half by then), beyond by swaps of 16 or 32 lanes of a wave, all without LDS and its latency.
struct Two {
    uint32_t a, b;
};
template <int O>
__device__ __forceinline__ Two both(uint32_t v) {
    if constexpr (O == 16) {
        const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        return {r[0], r[1]};
    } else if constexpr (O == 32) {
        const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        return {r[0], r[1]};
    } else {
        return {v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, O == 1 ? 0xB1 : O == 2 ? 0x4E : O == 4 ? 0x141 : 0x140, 0xf, 0xf, true)};
    }
}
// f over the L lanes of a team, the same in all of them; f(a, b) = f(b, a).
template <int L, int O = 1, class T, class F>
__device__ __forceinline__ T team(T v, F f) {
    if constexpr (O >= L) {
        return v;
    } else if constexpr (sizeof(T) == 8) {
        const uint64_t u = __builtin_bit_cast(uint64_t, v);
        const Two hi = both<O>((uint32_t)(u >> 32)), lo = both<O>((uint32_t)u);
        return team<L, 2 * O>(f(__builtin_bit_cast(T, (uint64_t)hi.a << 32 | lo.a), __builtin_bit_cast(T, (uint64_t)hi.b << 32 | lo.b)), f);
    } else {
        const Two r = both<O>(__builtin_bit_cast(uint32_t, v));
        return team<L, 2 * O>(f(__builtin_bit_cast(T, r.a), __builtin_bit_cast(T, r.b)), f);
    }
}
template <int L, class T>
__device__ __forceinline__ T team_max(T v) {
    return team<L>(v, [](T a, T b) { return a > b ? a : b; });
}
template <int L, class T>
__device__ __forceinline__ T team_min(T v) {
    return team<L>(v, [](T a, T b) { return a < b ? a : b; });
}
template <int L, class T>
__device__ __forceinline__ T team_sum(T v) {
    return team<L>(v, [](T a, T b) { return a + b; });
}

}  // namespace
}  // namespace j4q
