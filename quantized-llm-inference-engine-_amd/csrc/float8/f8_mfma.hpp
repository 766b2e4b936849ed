// The matrix instruction of the kernels in 8-bit floating point.
#pragma once

#include "../qcommon.hpp"

namespace llmopt {

typedef int i32x8 __attribute__((ext_vector_type(8)));

// acc += 128 products of numbers code x scale: 16 rows of `a` with 16 rows of `b`, lane l holding columns 32 (l / 16) .. of row l
// % 16 of both (any assignment of columns to lanes that is the same for both gives the same sums), and in byte A of scale_a
// (B of scale_b) the scale of that row (e8m0; byte 255 makes its sums NaN). Lane l gets rows 4 (l / 16) .. of a with row l % 16
// of b.
//
// The products of two codes are exact. The instruction adds the products of eight neighbouring columns first, and of these
// what is below 2^-13 of the largest is dropped (measured: 2^16 + 2^2 loses the second term in a group of eight, 2^16 + 2^-9
// keeps it across two groups; v_mfma_f32_16x16x32_fp8_fp8 does the same, the bf16 instructions do not); beyond that the
// sums are fp32. A sum is off by at most 7 * 2^-13 of the largest products' magnitudes added up. Measured, of its typical size: 1.5e-5 for
// channels of like strength, 2.7e-5 where 1 % of them are 8 times as strong, 8e-5 at 0.2 % 100 times, at most 1e-4 where a few are
// nearly all of a sum; a rounding to fp16 brings 2e-4, one to bf16 1.7e-3. The bf16 instructions on the same codes would be
// exact to fp32 at less than half the rate.
template <int A = 0, int B = 0>
__device__ __forceinline__ f32x4 mfma_f8(i32x8 a, i32x8 b, f32x4 acc, uint32_t scale_a, uint32_t scale_b) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc, 0, 0, A, int(scale_a), B, int(scale_b));
}

}  // namespace llmopt
