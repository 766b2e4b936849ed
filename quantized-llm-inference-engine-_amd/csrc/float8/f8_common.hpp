// Shared by the kernels of the decoder's steps in 8-bit floating point (llmopt_float8.h): argument blocks, and the
// quantizing of a group of 128 numbers.
#pragma once

#include <type_traits>

#include "../qcommon.hpp"

namespace llmopt {

constexpr int kF8Group = 128;       // columns of a scale, and rows of a weight's

struct F8QuantArgs {
  const void* x;  // [rows, cols]
  int64_t ldx;
  uint8_t* codes;
  int64_t ldc;
  uint8_t* scales;
  int64_t lds;
  int64_t rows, cols;
  int vec;  // x's rows 16-byte aligned, the codes' 8-byte, and cols a multiple of 8
};

struct F8NormArgs {
  const void* x;
  int64_t ldx;
  const void* residual;  // null: none
  int64_t ldr;
  void* h_out;
  int64_t ldh;
  const void* weight;
  uint8_t* codes;
  int64_t ldc;
  uint8_t* scales;
  int64_t lds;
  int64_t rows, hidden;
  float eps;
  int vec;  // all rows 16-byte aligned, the codes' 8-byte, and hidden a multiple of 8
};

// A weight [N, K] of codes.
struct F8Weight {
  const uint8_t* codes;
  int64_t ld;
  const uint8_t* scales;  // [ceil(N / 128), ceil(K / 128)]
  int64_t lds;
};

// silu(gate) * up of fp32 sums, quantized by rows.
struct F8ActArgs {
  const float* gate;  // [rows, cols], rows of `ld` elements; up likewise
  const float* up;
  int64_t ld;
  uint8_t* codes;
  int64_t ldc;
  uint8_t* scales;
  int64_t lds;
  int64_t rows, cols;
};

// Products of x [M, K] with weights [N, K]: y = x w[0]^T + bias, or silu(x w[0]^T) * (x w[1]^T) quantized where w[1] has codes.
// For the tiled kernels all rows of codes are 16-byte aligned, K is a multiple of 16, and the strides are at most 2^21.
struct F8TilesArgs {
  const uint8_t* x;
  int64_t ldx;
  const uint8_t* x_scales;
  int64_t ldxs;
  F8Weight w[2];
  const void* bias;
  void* y;
  int64_t ldy;
  uint8_t* codes;
  int64_t ldc;
  uint8_t* scales;
  int64_t lds;
  int64_t M, N, K;
  int vec;  // the output's rows are 16-byte aligned
  int steps;
  uint32_t tiles_n, tiles_m;         // (set by the launch)
  uint32_t splits, steps_per_split;  // of K over workgroups
  float* parts;                      // splits > 1: [splits][M][ld_parts]
  int64_t ld_parts;
};

// A workgroup's tile: weight rows x tokens.
enum class F8Shape { k256x256, k256x128, k256x64, k128x128, k128x64 };

// The kernel of at most 16 tokens; operands as in F8TilesArgs. With a second weight its product's rows come in y behind the
// first one's (and there is no bias).
struct F8DecodeArgs {
  const uint8_t* x;
  int64_t ldx;
  const uint8_t* x_scales;
  int64_t ldxs;
  F8Weight w[2];
  const void* bias;
  void* y;
  int64_t ldy;
  int64_t M, N, K;
  uint32_t steps, tiles;  // (set by the launch)
};

hipError_t launch_f8_quantize(const F8QuantArgs& a, int dtype, int64_t block_rows, hipStream_t stream);
hipError_t launch_f8_rmsnorm(const F8NormArgs& a, int dtype, hipStream_t stream);
hipError_t launch_f8_act(const F8ActArgs& a, hipStream_t stream);
hipError_t launch_f8_tiles(const F8TilesArgs& a, F8Shape shape, int out_dtype, hipStream_t stream);
// The sum of `splits` (2, 4 or 8) parts [M, ld_parts] in their order, plus the bias, rounded into y.
struct F8JoinArgs {
  const float* parts;
  uint32_t splits;
  int64_t M, N, ld_parts;  // (a multiple of 16)
  const void* bias;
  void* y;
  int64_t ldy;
};
hipError_t launch_f8_join(const F8JoinArgs& a, int out_dtype, hipStream_t stream);
hipError_t launch_f8_decode(F8DecodeArgs a, int out_dtype, hipStream_t stream);
// Rows of any alignment; the gated product where w[1] has codes. (The other kernels' sizes are not set.)
hipError_t launch_f8_any(const F8TilesArgs& a, int out_dtype, hipStream_t stream);

// ---- groups -----------------------------------------------------------------------------------------

template <int CTRL>
__device__ __forceinline__ uint32_t dpp_max(uint32_t v) {
  return max(v, uint32_t(__builtin_amdgcn_update_dpp(0, int(v), CTRL, 0xF, 0xF, true)));
}

// The largest of 16 neighbouring lanes, in all of them: pairs, quads, mirrored halves of 8 and of 16 lanes.
__device__ __forceinline__ uint32_t max16(uint32_t v) {
  v = dpp_max<0xB1>(v);   // quad_perm 1 0 3 2
  v = dpp_max<0x4E>(v);   // quad_perm 2 3 0 1
  v = dpp_max<0x141>(v);  // row_half_mirror
  return dpp_max<0x140>(v);  // row_mirror
}

// Magnitudes are compared as the whole numbers of their bits: infinities and NaN are above every finite one.
__device__ __forceinline__ uint32_t magnitude(float f) { return __float_as_uint(f) & 0x7FFFFFFFu; }

// The scale 2^e that a group of magnitudes up to amax needs, as e + 127: the smallest e >= -127 with amax <= 448 2^e. 448 is
// 1.75 2^8, so e is amax's exponent less 8, one more where its fraction is above 1.75. 255 (NaN) for what is not finite.
__device__ __forceinline__ uint32_t f8_scale(uint32_t amax_bits) {
  const uint32_t e = (amax_bits + 0x1FFFFFu) >> 23;
  return amax_bits >= 0x7F800000u ? 255u : e > 8u ? e - 8u : 0u;
}

// 2^-e of a scale that f8_scale gave (at most 2^120, so this is no subnormal number); 0 for NaN.
__device__ __forceinline__ float f8_inverse(uint32_t scale) { return scale == 255u ? 0.0f : __uint_as_float((254u - scale) << 23); }

// Codes of four numbers: the products are exact and at most 448 (but for tiny ones, below every code); zeros in a group that
// is not finite.
__device__ __forceinline__ uint32_t f8_codes4(float a, float b, float c, float d, float inv) {
  if (inv == 0.0f) return 0u;
  const int w = __builtin_amdgcn_cvt_pk_fp8_f32(a * inv, b * inv, 0, false);
  return uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(c * inv, d * inv, w, true));
}

// silu(gate) * up in fp32, with the hardware's exponential and reciprocal (a step of fp32 each; 2^-22 |gate| of the
// exponential's argument). Far below zero the exponential is infinite and the product 0.
__device__ __forceinline__ float f8_swiglu(float gate, float up) {
  return gate * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(gate * -1.44269504f)) * up;
}

// Two numbers as 16-bit ones, to nearest, ties to even.
template <class Out>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  if constexpr (Out::id == kDtBf16) {
    const f32x2 v = {lo, hi};
    typedef __bf16 pair __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, pair));
  } else {
    return uint32_t(Out::store(lo)) | (uint32_t(Out::store(hi)) << 16);
  }
}

// Eight neighbouring numbers of a row, from column c on; zeros behind `cols`.
template <class Act>
__device__ __forceinline__ void load8(const typename Act::raw* row, int64_t c, int64_t cols, bool vec, float* v) {
  if (vec && c < cols) {
    if constexpr (sizeof(typename Act::raw) == 4) {
      const f32x4 lo = *reinterpret_cast<const f32x4*>(row + c), hi = *reinterpret_cast<const f32x4*>(row + c + 4);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = lo[i], v[4 + i] = hi[i];
    } else {
      const u32x4 w = *reinterpret_cast<const u32x4*>(row + c);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[2 * i] = Act::load(typename Act::raw(w[i] & 0xFFFFu));
        v[2 * i + 1] = Act::load(typename Act::raw(w[i] >> 16));
      }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = c + i < cols ? Act::load(row[c + i]) : 0.0f;
}

__device__ __forceinline__ void store_codes8(uint8_t* row, int64_t c, int64_t cols, bool vec, u32x2 w) {
  if (vec) {
    if (c < cols) __builtin_nontemporal_store(w, reinterpret_cast<u32x2*>(row + c));
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (c + i < cols) row[c + i] = uint8_t(w[i >> 2] >> (8 * (i & 3)));
}

// Quantizes a row's numbers, eight per lane (16 neighbouring lanes hold a group, and all of them call this).
__device__ __forceinline__ void quantize8(const float* v, uint8_t* codes, uint8_t* scales, int64_t c, int64_t cols, bool vec) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, magnitude(v[i]));
  const uint32_t s = f8_scale(max16(top));
  const float inv = f8_inverse(s);
  store_codes8(codes, c, cols, vec, u32x2{f8_codes4(v[0], v[1], v[2], v[3], inv), f8_codes4(v[4], v[5], v[6], v[7], inv)});
  if ((threadIdx.x & 15) == 0 && c < cols) scales[c / kF8Group] = uint8_t(s);
}

}  // namespace llmopt
