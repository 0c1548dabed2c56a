// Loads of weights for the matrix cores and exchanges between the lane groups of a wave (lanes 16 g .. 16 g + 15), for kernels in
// which a lane loads 16 contiguous bytes of a row (gemv_mfma.h, experts_few.hip).
#pragma once

#include "gemv_impl.h"

namespace j4q {
namespace gmf {

using gemv::f32x4;
using gemv::kOob;
using gemv::make_rsrc;
using gemv::Rsrc;
using gemv::u32x2;
using gemv::u32x4;

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

// Weight loads keep the default cache policy, unlike the batch-1 kernel's non-temporal
// stream: a wave's item covers 64 bytes of each of 16 rows, half of a 128-byte line, and
// its next item the other half, which a non-temporal load fetched again (measured: B = 16
// decode step 2.64 -> 2.45 ms).
constexpr int kTile = 0;
// A load that is not `ok` takes the out-of-range lane offset (the scalar offset stays
// unconditional). The lane offset passes through an empty asm: with a select on the tile's
// liveness visible in the scalar offset, the compiler split some loads into two branches,
// and the wait counts it then derived waited for loads issued after the ones needed.
__device__ __forceinline__ uint32_t lane_off(uint32_t vo, bool ok) {
    uint32_t v = ok ? vo : kOob;
    asm("" : "+v"(v));
    return v;
}
__device__ __forceinline__ u32x4 ld128(__amdgpu_buffer_rsrc_t r, uint32_t vo, uint32_t so, bool ok) {
    return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, lane_off(vo, ok), so, kTile));
}
__device__ __forceinline__ u32x2 ld64(__amdgpu_buffer_rsrc_t r, uint32_t vo, uint32_t so, bool ok) {
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(r, lane_off(vo, ok), so, kTile));
}
__device__ __forceinline__ uint32_t ld32(__amdgpu_buffer_rsrc_t r, uint32_t vo, uint32_t so, bool ok) {
    return (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(r, lane_off(vo, ok), so, kTile);
}
__device__ __forceinline__ uint32_t ld16(__amdgpu_buffer_rsrc_t r, uint32_t vo, uint32_t so, bool ok) {
    return (uint32_t)__builtin_amdgcn_raw_buffer_load_b16(r, lane_off(vo, ok), so, kTile);
}

// On entry lane group g (lanes 16g..16g+15) holds v[0..3] = dwords 0..3 of its own unit g;
// on exit v[t] holds dword g of unit t.
__device__ __forceinline__ void xpose4(uint32_t (&v)[4]) {
    const auto a = __builtin_amdgcn_permlane32_swap(v[0], v[2], false, false);
    const auto b = __builtin_amdgcn_permlane32_swap(v[1], v[3], false, false);
    const auto c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
    const auto d = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
    v[0] = c[0];
    v[1] = c[1];
    v[2] = d[0];
    v[3] = d[1];
}

// o[t] = x of lane group t (same lane within the group), in every lane.
__device__ __forceinline__ void bcast4(float x, float (&o)[4]) {
    const uint32_t v = __builtin_bit_cast(uint32_t, x);
    const auto a = __builtin_amdgcn_permlane32_swap(v, v, false, false);  // [g0 g1 g0 g1], [g2 g3 g2 g3]
    const auto b0 = __builtin_amdgcn_permlane16_swap(a[0], a[0], false, false);
    const auto b1 = __builtin_amdgcn_permlane16_swap(a[1], a[1], false, false);
    o[0] = __builtin_bit_cast(float, (uint32_t)b0[0]);
    o[1] = __builtin_bit_cast(float, (uint32_t)b0[1]);
    o[2] = __builtin_bit_cast(float, (uint32_t)b1[0]);
    o[3] = __builtin_bit_cast(float, (uint32_t)b1[1]);
}

}  // namespace gmf
}  // namespace j4q
