// y = x w^T + bias of codes with block scales, for rows of any length, stride and alignment: the kernel of shapes that the
// tiled ones do not take.
//
// A wave multiplies 16 rows of the weight with 16 tokens, a group of 128 columns at a time (mfma_f8).
#include "f8_common.hpp"
#include "f8_mfma.hpp"

namespace llmopt {
namespace {

// 32 codes of a row from column k on, zeros behind its end; no alignment is asked for.
__device__ __forceinline__ i32x8 load32(const uint8_t* row, int64_t k, int64_t K) {
  i32x8 v = {0, 0, 0, 0, 0, 0, 0, 0};
  if (k + 32 <= K) {
    __builtin_memcpy(&v, row + k, 32);
    return v;
  }
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    const uint32_t byte = k + i < K ? row[k + i] : 0u;
    v[i >> 2] |= int(byte << (8 * (i & 3)));
  }
  return v;
}

template <class Out>
__global__ void __launch_bounds__(256) linear_any_kernel(const F8LinearArgs a, uint32_t token_tiles) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t nb = blockIdx.x / token_tiles;
  const int64_t n0 = (int64_t(nb) * 4 + wave) * 16, m0 = int64_t(blockIdx.x - nb * token_tiles) * 16;
  if (n0 >= a.N) return;
  const int r = lane & 15, g = lane >> 4;
  const int64_t m = m0 + r, mr = m < a.M ? m : a.M - 1, nr = n0 + r < a.N ? n0 + r : a.N - 1;
  const uint8_t* xr = a.x + mr * a.ldx;
  const uint8_t* wr = a.w.codes + nr * a.w.ld;
  const uint8_t* xs = a.x_scales + mr * a.ldxs;
  const uint8_t* ws = a.w.scales + (n0 / kF8Group) * a.w.lds;
  f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int64_t k = 0; k < a.K; k += kF8Group) {
    const i32x8 wv = load32(wr, k + 32 * g, a.K), xv = load32(xr, k + 32 * g, a.K);
    acc = mfma_f8(wv, xv, acc, ws[k / kF8Group], xs[k / kF8Group]);
  }
  if (m >= a.M) return;
  auto* y = static_cast<typename Out::raw*>(a.y) + m * a.ldy;
  const auto* bias = static_cast<const typename Out::raw*>(a.bias);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t n = n0 + 4 * g + i;
    if (n < a.N) y[n] = Out::store(bias ? acc[i] + Out::load(bias[n]) : acc[i]);
  }
}

}  // namespace

hipError_t launch_f8_linear_any(const F8LinearArgs& a, int out_dtype, hipStream_t stream) {
  if (a.M == 0 || a.N == 0) return hipSuccess;
  const int64_t tiles = (a.M + 15) / 16;
  const dim3 grid(unsigned(tiles * ((a.N + 63) / 64)));
  if (out_dtype == kDtF32)
    hipLaunchKernelGGL(linear_any_kernel<ActF32>, grid, dim3(256), 0, stream, a, uint32_t(tiles));
  else if (out_dtype == kDtF16)
    hipLaunchKernelGGL(linear_any_kernel<ActF16>, grid, dim3(256), 0, stream, a, uint32_t(tiles));
  else
    hipLaunchKernelGGL(linear_any_kernel<ActBf16>, grid, dim3(256), 0, stream, a, uint32_t(tiles));
  return hipGetLastError();
}

}  // namespace llmopt
