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

// What the gated product reads: x [M, K] and two weights [N, K].
struct F8Gated {
  const uint8_t* x;
  int64_t ldx;
  const uint8_t* x_scales;
  int64_t ldxs;
  F8Weight w[2];
  int64_t K;
};

// silu(gate) * up of fp32 sums, quantized by rows.
struct F8ActArgs {
  F8Gated in;  // of which they are the sums
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
  int steps;
  uint32_t tiles_n, tiles_m;         // (set by the launch)
  uint32_t splits, steps_per_split;  // of K over workgroups
  float* parts;                      // splits > 1: [splits][M][ld_parts]
  int64_t ld_parts;
};

// A workgroup's tile: weight rows x tokens.
enum class F8Shape { k256x256, k256x128, k256x64, k128x128, k128x64 };

// The kernel of few tokens; operands as in F8TilesArgs. With a second weight its product's rows come in y behind the
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
// exponential's argument). Below -87.3 the reciprocal is less than the least normal number and the product 0, which is off by 2^-119 |up|.
__device__ __forceinline__ float f8_swiglu(float gate, float up) {
  return gate * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(gate * -1.44269504f)) * up;
}

// ---- maxima next to a border of the scales -------------------------------------------------------------

// A group's scale doubles where its largest magnitude passes 1.75 2^i, and the matrix cores' sums (f8_mfma.hpp) would put some groups
// on the wrong side. So a maximum within 2^-10 of a border, one in some 350, is taken once more, from fp32 sums of exact products of
// the numbers that it may be. (A number that stays a little above 448 2^e rounds to that.)
// 2^-10 is more than a sum of which one product is nearly all can be off by, seven times 2^-13 of it; other sums are off by less,
// as the bits dropped from many products go either way. How far maxima of silu(gate) * up are off, measured (MI355X, K of 512, 1024
// and 4096, 50,000 to 100,000 groups each): channels of like strength 1.3e-5 rms, 1 % of them 8 times as strong 2.5e-5, 0.2 % 100
// times 8e-5, one or two 1000 times and more 1.2e-4; the largest of a million 8.6e-4. Without this 3 to 13 groups in 100,000
// would be on the wrong side, with a window of 1e-4 none of the first, but up to 8 of the last.
// Measured (MI355X, in a graph, us, without / a window of 1e-4 with a walk for each number / as it is; gate and up of 14336 x 4096): 4
// tokens 24.1 / 24.3 / 25.1, 200 tokens 35 / 38 / 38.5, 8192 tokens 750 / 772 / 797; 2816 x 1024, 8192 tokens 58 / 65 / 72: half of
// that for the walks, of some 3 us each, half for the registers that they take.
constexpr uint32_t kF8Near = 14336;  // in steps of the fraction's 23 bits
__device__ __forceinline__ bool f8_near(uint32_t bits) {
  return bits < 0x7F800000u && ((bits - 0x600000u + kF8Near) & 0x7FFFFFu) < 2 * kF8Near;
}

// 16 codes of a row from column k on, zeros behind its end. ANY: of any alignment and length.
template <bool ANY>
__device__ __forceinline__ u32x4 load_codes16(const uint8_t* row, int64_t k, int64_t K) {
  u32x4 v = {0, 0, 0, 0};
  if constexpr (ANY) {
    for (int i = 0; i < 16 && k + i < K; ++i) v[i >> 2] |= uint32_t(row[k + i]) << (8 * (i & 3));
  } else {
    if (k < K) v = *reinterpret_cast<const u32x4*>(row + k);
  }
  return v;
}

// Token m's feature n, by a whole wave (m and n the same in all its lanes): 4096 columns at a time, all their loads at once.
template <bool ANY>
__device__ __forceinline__ float f8_gated_again(const F8Gated& in, int64_t m, int64_t n) {
  float sum[2] = {0.0f, 0.0f};
  const uint8_t* rows[3] = {in.x + m * in.ldx, in.w[0].codes + n * in.w[0].ld, in.w[1].codes + n * in.w[1].ld};
  const uint8_t* scales[3] = {in.x_scales + m * in.ldxs, in.w[0].scales + n / kF8Group * in.w[0].lds, in.w[1].scales + n / kF8Group * in.w[1].lds};
#pragma unroll 1
  for (int64_t base = 16 * (threadIdx.x & 63); base < in.K; base += 4096) {
    u32x4 c[4][3];
    int e[4][3];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t k = base + 1024 * j;
#pragma unroll
      for (int t = 0; t < 3; ++t) {
        c[j][t] = load_codes16<ANY>(rows[t], k, in.K);
        e[j][t] = scales[t][k < in.K ? k / kF8Group : 0];
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float dot[2] = {0.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f32x2 x0 = __builtin_amdgcn_cvt_pk_f32_fp8(int(c[j][0][i]), false), x1 = __builtin_amdgcn_cvt_pk_f32_fp8(int(c[j][0][i]), true);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const f32x2 w0 = __builtin_amdgcn_cvt_pk_f32_fp8(int(c[j][1 + t][i]), false), w1 = __builtin_amdgcn_cvt_pk_f32_fp8(int(c[j][1 + t][i]), true);
          dot[t] = __builtin_fmaf(x0[0], w0[0], __builtin_fmaf(x0[1], w0[1], dot[t]));
          dot[t] = __builtin_fmaf(x1[0], w1[0], __builtin_fmaf(x1[1], w1[1], dot[t]));
        }
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) sum[t] += __builtin_ldexpf(dot[t], e[j][0] + e[j][1 + t] - 254);
    }
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    sum[0] += __shfl_xor(sum[0], off, 64);
    sum[1] += __shfl_xor(sum[1], off, 64);
  }
  return f8_swiglu(sum[0], sum[1]);
}

// A wave's walks for one tile, at most: some 3 us each, about as long as the tile itself. Numbers drawn at random next to a
// border are one or two of a wave. More than 16 that differ come of features that are equal; what is not walked then keeps the scale that
// the matrix cores' sums give.
constexpr int kF8Walks = 16;

// For a whole wave of lanes that hold V neighbouring features from n on of U tokens, 16 apart from their m on. Lanes that agree in the
// bits of SAME have the same tokens; top is the largest magnitude of a token's features in them (0 behind the last token), and
// exact when this returns, where a border is near. Tokens whose V numbers agree in a 32-bit hash of their bits are taken for equal,
// and walked once: a batch of one token over and over is next to a border as a whole (4096 such tokens by 8192 x 1024 take 99 us, with a
// walk each 569, other tokens 83).
template <bool ANY, int SAME, class In, int U, int V>
__device__ __forceinline__ void f8_settle(In&& inputs, const float (&v)[U][V], uint32_t (&top)[U], int64_t m, int64_t n) {
  static_assert(U * V <= 64, "a bit for each number");
  bool any = false;
#pragma unroll
  for (int u = 0; u < U; ++u) any |= f8_near(top[u]);
  if (__builtin_expect_with_probability(__ballot(any) == 0, 1, 0.999)) return;
  const F8Gated in = inputs();
  uint32_t pending[2] = {0, 0}, exact[U] = {}, hash[U] = {};
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t below = f8_near(top[u]) ? top[u] - 2 * kF8Near - 1 : 0x7FFFFFFFu;
#pragma unroll
    for (int i = 0; i < V; ++i) {  // (a sign rather than a comparison, which would hold scalar registers)
      pending[(u * V + i) / 32] |= ((below - magnitude(v[u][i])) >> 31) << ((u * V + i) % 32);
      hash[u] = (hash[u] << 5 | hash[u] >> 27) + __float_as_uint(v[u][i]) * 0x9E3779B1u;
    }
  }
  const int own = threadIdx.x & 63;
  uint64_t mask = __ballot((pending[0] | pending[1]) != 0);
#pragma unroll 1
  for (int walk = 0; walk < kF8Walks && mask != 0; ++walk) {
    const int lane = __builtin_ctzll(mask);
    auto of_lane = [&](uint32_t value) { return uint32_t(__builtin_amdgcn_readlane(int(value), lane)); };
    auto of_lane64 = [&](int64_t value) { return int64_t(uint64_t(of_lane(uint32_t(value >> 32))) << 32 | of_lane(uint32_t(value))); };
    const uint32_t lo = of_lane(pending[0]);
    const int at = lo ? __builtin_ctz(lo) : 32 + __builtin_ctz(of_lane(pending[1]));
    const int64_t first = of_lane64(n);
    const uint32_t again = magnitude(f8_gated_again<ANY>(in, of_lane64(m) + at / V * 16, first + at % V));
    uint32_t key = 0;
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (at / V == u) key = of_lane(hash[u]);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool equal = n == first && hash[u] == key;
      const uint64_t lanes = __ballot(equal);  // of this feature: at most one of a token
      if (lanes >> ((lane & ~SAME) | (own & SAME)) & 1) exact[u] = max(exact[u], again);
      if (equal) pending[(u * V + at % V) / 32] &= ~(1u << ((u * V + at % V) % 32));
    }
    mask = __ballot((pending[0] | pending[1]) != 0);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    bool all = true;  // of the token's numbers, walked
    if (mask != 0) {
      constexpr uint64_t kToken = SAME == 15 ? 0x0001000100010001u : 0xFFFFu;
      static_assert(SAME == 15 || SAME == 48, "the lanes of a token");
      const uint64_t left = __ballot(((uint64_t(pending[1]) << 32 | pending[0]) >> (u * V) & ((uint64_t(1) << (V - 1) << 1) - 1)) != 0);
      all = (left & (kToken << (own & SAME))) == 0;
    }
    if (f8_near(top[u]) && all) top[u] = exact[u];
  }
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

// The largest magnitude of eight numbers per lane of 16 neighbouring lanes, in all of them.
__device__ __forceinline__ uint32_t largest8(const float* v) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, magnitude(v[i]));
  return max16(top);
}

// Quantizes a row's numbers, eight per lane (16 neighbouring lanes hold a group, and all of them call this).
__device__ __forceinline__ void quantize8(const float* v, uint32_t top, uint8_t* codes, uint8_t* scales, int64_t c, int64_t cols, bool vec) {
  const uint32_t s = f8_scale(top);
  const float inv = f8_inverse(s);
  store_codes8(codes, c, cols, vec, u32x2{f8_codes4(v[0], v[1], v[2], v[3], inv), f8_codes4(v[4], v[5], v[6], v[7], inv)});
  if ((threadIdx.x & 15) == 0 && c < cols) scales[c / kF8Group] = uint8_t(s);
}
__device__ __forceinline__ void quantize8(const float* v, uint8_t* codes, uint8_t* scales, int64_t c, int64_t cols, bool vec) {
  quantize8(v, largest8(v), codes, scales, c, cols, vec);
}

}  // namespace llmopt
