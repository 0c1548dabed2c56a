// Checks of caller memory that entry points share.
#pragma once

#include <stdint.h>

#include "jax4j_mi355x.h"

namespace j4q {

inline bool aligned(const void *p, uintptr_t a) { return ((uintptr_t)p & (a - 1)) == 0; }

inline bool dense_type(int t) { return t == J4Q_KIND_F32 || t == J4Q_KIND_BF16; }
inline int64_t dense_size(int t) { return t == J4Q_KIND_BF16 ? 2 : 4; }

// Whether two tensors of `rows` rows, strides and widths in bytes, share a byte.
inline bool overlap(const void *a, int64_t a_stride, int64_t a_width, const void *b, int64_t b_stride, int64_t b_width, int64_t rows) {
    const uintptr_t a0 = (uintptr_t)a, b0 = (uintptr_t)b;
    if (a0 >= b0 + (rows - 1) * b_stride + b_width || b0 >= a0 + (rows - 1) * a_stride + a_width) return false;
    if (a_stride != b_stride) return true;
    const int64_t between = (int64_t)(b0 - a0) % a_stride, at = between < 0 ? between + a_stride : between;  // windows of the same rows
    return at < a_width || at + b_width > a_stride;
}

// Whether two ranges of bytes share one.
inline bool overlap(const void *a, uint64_t a_bytes, const void *b, uint64_t b_bytes) {
    return (uintptr_t)a < (uintptr_t)b + b_bytes && (uintptr_t)b < (uintptr_t)a + a_bytes;
}

}  // namespace j4q
