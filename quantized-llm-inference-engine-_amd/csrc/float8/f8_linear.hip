// Products of rows of any length, stride and alignment: the kernels of shapes that the others do not take. A wave multiplies 16
// rows of the weight with 16 tokens, a group of 128 columns at a time, straight from memory. Bound by those loads, of which no two waves
// share any, and of rows that start at any byte as pieces of several lines: 4096 x 14330 takes 87 us of one token, 149 of 32 and 18 ms of
// 8192 (MI355X), 7, 9 and 47 times what rows of whole 16 bytes do (4096 x 14336 with the tokens' rows alone at an odd address 60, 65 and
// 7.1 ms). A layer's weights and activations are aligned.
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

// acc[t] += 16 rows of weight t from n0 on times 16 tokens from m0 on; rows and tokens behind the last repeat it.
template <int W>
__device__ __forceinline__ void sums_any(const F8TilesArgs& a, int64_t n0, int64_t m0, f32x4 (&acc)[W]) {
  const int r = threadIdx.x & 15, g = (threadIdx.x & 63) >> 4;
  const int64_t m = m0 + r < a.M ? m0 + r : a.M - 1, n = n0 + r < a.N ? n0 + r : a.N - 1;
  const uint8_t* xr = a.x + m * a.ldx;
  const uint8_t* xs = a.x_scales + m * a.ldxs;
#pragma unroll
  for (int t = 0; t < W; ++t) acc[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  for (int64_t k = 0; k < a.K; k += kF8Group) {
    const i32x8 xv = load32(xr, k + 32 * g, a.K);
    const uint32_t sx = xs[k / kF8Group];
#pragma unroll
    for (int t = 0; t < W; ++t)
      acc[t] = mfma_f8(load32(a.w[t].codes + n * a.w[t].ld, k + 32 * g, a.K), xv, acc[t],
                       a.w[t].scales[(n0 / kF8Group) * a.w[t].lds + k / kF8Group], sx);
  }
}

template <class Out>
__global__ void __launch_bounds__(256) linear_any_kernel(const F8TilesArgs a, uint32_t token_tiles) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t nb = blockIdx.x / token_tiles;
  const int64_t n0 = (int64_t(nb) * 4 + wave) * 16, m0 = int64_t(blockIdx.x - nb * token_tiles) * 16;
  if (n0 >= a.N) return;
  f32x4 acc[1];
  sums_any<1>(a, n0, m0, acc);
  const int64_t m = m0 + (lane & 15);
  if (m >= a.M) return;
  auto* y = static_cast<typename Out::raw*>(a.y) + m * a.ldy;
  const auto* bias = static_cast<const typename Out::raw*>(a.bias);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t n = n0 + 4 * (lane >> 4) + i;
    if (n < a.N) y[n] = Out::store(bias ? acc[0][i] + Out::load(bias[n]) : acc[0][i]);
  }
}

// A workgroup takes a group of 128 features, a wave 16 of them.
__global__ void __launch_bounds__(512) gated_any_kernel(const F8TilesArgs a, uint32_t token_tiles) {
  __shared__ uint32_t tops[8][16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
  const uint32_t nb = blockIdx.x / token_tiles;
  const int64_t n0 = int64_t(nb) * kF8Group + 16 * wave, m0 = int64_t(blockIdx.x - nb * token_tiles) * 16;
  float v[1][4] = {{0.0f, 0.0f, 0.0f, 0.0f}};
  uint32_t top = 0;
  if (n0 < a.N) {
    f32x4 acc[2];
    sums_any<2>(a, n0, m0, acc);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n0 + 4 * g + i < a.N && m0 + r < a.M) v[0][i] = f8_swiglu(acc[0][i], acc[1][i]);
    uint32_t most[1] = {0};
#pragma unroll
    for (int i = 0; i < 4; ++i) most[0] = max(most[0], magnitude(v[0][i]));
    most[0] = max(most[0], uint32_t(__shfl_xor(int(most[0]), 16, 64)));
    most[0] = max(most[0], uint32_t(__shfl_xor(int(most[0]), 32, 64)));
    f8_settle<true, 15>([&] { return F8Gated{a.x, a.ldx, a.x_scales, a.ldxs, {a.w[0], a.w[1]}, a.K}; }, v, most, m0 + r, n0 + 4 * g);
    top = most[0];
  }
  if (g == 0) tops[wave][r] = top;
  __syncthreads();
  const int64_t m = m0 + r;
  if (m >= a.M) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, tops[i][r]);
  const uint32_t scale = f8_scale(top), codes = f8_codes4(v[0][0], v[0][1], v[0][2], v[0][3], f8_inverse(scale));
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (n0 + 4 * g + i < a.N) a.codes[m * a.ldc + n0 + 4 * g + i] = uint8_t(codes >> (8 * i));
  if (wave == 0 && g == 0) a.scales[m * a.lds + nb] = uint8_t(scale);
}

}  // namespace

hipError_t launch_f8_any(const F8TilesArgs& a, int out_dtype, hipStream_t stream) {
  const int64_t tiles = (a.M + 15) / 16;
  if (a.w[1].codes) {
    const dim3 grid(unsigned(tiles * ((a.N + kF8Group - 1) / kF8Group)));
    hipLaunchKernelGGL(gated_any_kernel, grid, dim3(512), 0, stream, a, uint32_t(tiles));
    return hipGetLastError();
  }
  const dim3 grid(unsigned(tiles * ((a.N + 63) / 64)));
  if (out_dtype == kDtF16)
    hipLaunchKernelGGL(linear_any_kernel<ActF16>, grid, dim3(256), 0, stream, a, uint32_t(tiles));
  else
    hipLaunchKernelGGL(linear_any_kernel<ActBf16>, grid, dim3(256), 0, stream, a, uint32_t(tiles));
  return hipGetLastError();
}

}  // namespace llmopt
