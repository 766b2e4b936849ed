// The products of few tokens: bound by the weight's bytes, which go from memory straight into the matrix core's operands.
//
// A wave multiplies RT tiles of 16 weight rows with TM tiles of 16 tokens. Steps of 128 columns are dealt to the waves of a
// workgroup in turn (and to `splits` workgroups in runs), so that together they read whole kilobytes of each row; every wave
// has the operands of DEPTH steps on their way. The waves' sums are added in LDS in a fixed order.
#include "f8_common.hpp"
#include "f8_mfma.hpp"

namespace llmopt {
namespace {

constexpr uint32_t kOutside = 0x7FFFFFF0u;

// One wave's walk over its steps: acc[t][u] += weight tile t times token tile u. `w` holds the tiles' buffers and row offsets.
template <int RT, int TM, int DEPTH>
struct Walk {
  __amdgpu_buffer_rsrc_t wq[RT], ws[RT], xq, xs;
  uint32_t w_off[RT], x_off[TM], xs_off[TM];  // this lane's rows
  uint32_t K, steps;

  struct Slot {
    u32x4 w[RT][2], x[TM][2];
    uint32_t sw[RT], sx[TM];
  };

  // Lane (r, g) takes the 16-byte pieces g and g + 4 of its row's 128 columns; what lies behind the end reads as zeros.
  __device__ __forceinline__ void load(Slot& s, uint32_t step, uint32_t end, int g) const {
    const uint32_t k = step * kF8Group + 16 * g;
    const bool live = step < end, lo = live && k < K, hi = live && k + 64 < K;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      s.w[t][0] = __builtin_amdgcn_raw_buffer_load_b128(wq[t], int(lo ? w_off[t] + k : kOutside), 0, 0);
      s.w[t][1] = __builtin_amdgcn_raw_buffer_load_b128(wq[t], int(hi ? w_off[t] + k + 64 : kOutside), 0, 0);
      s.sw[t] = __builtin_amdgcn_raw_buffer_load_b8(ws[t], int(live ? step : kOutside), 0, 0);
    }
#pragma unroll
    for (int u = 0; u < TM; ++u) {
      s.x[u][0] = __builtin_amdgcn_raw_buffer_load_b128(xq, int(lo ? x_off[u] + k : kOutside), 0, 0);
      s.x[u][1] = __builtin_amdgcn_raw_buffer_load_b128(xq, int(hi ? x_off[u] + k + 64 : kOutside), 0, 0);
      s.sx[u] = __builtin_amdgcn_raw_buffer_load_b8(xs, int(live ? xs_off[u] + step : kOutside), 0, 0);
    }
  }

  // Steps first, first + stride, ... below end.
  __device__ __forceinline__ void run(uint32_t first, uint32_t stride, uint32_t end, f32x4 (&acc)[RT][TM]) const {
    const int g = (threadIdx.x & 63) >> 4;
    Slot slot[DEPTH];
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) load(slot[d], first + d * stride, end, g);
    for (uint32_t s = first; s < end; s += DEPTH * stride) {
#pragma unroll
      for (int d = 0; d < DEPTH; ++d) {
        Slot& now = slot[d];
        i32x8 w[RT], x[TM];
#pragma unroll
        for (int t = 0; t < RT; ++t)
          w[t] = __builtin_bit_cast(i32x8, __builtin_shufflevector(now.w[t][0], now.w[t][1], 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
        for (int u = 0; u < TM; ++u)
          x[u] = __builtin_bit_cast(i32x8, __builtin_shufflevector(now.x[u][0], now.x[u][1], 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
          for (int u = 0; u < TM; ++u) acc[t][u] = mfma_f8(w[t], x[u], acc[t][u], now.sw[t], now.sx[u]);
        load(now, s + (DEPTH + d) * stride, end, g);
      }
    }
  }
};

// y of 16 RT features and M <= 16 TM tokens, or this split's part of it.
template <int RT, int TM, int WAVES, int DEPTH, class Out>
__global__ void __launch_bounds__(64 * WAVES) decode_kernel(const F8DecodeArgs a) {
  __shared__ __align__(16) float sums[WAVES][RT * TM][64][4];
  const int lane = threadIdx.x & 63;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;
  const uint32_t split = a.splits > 1 ? __builtin_amdgcn_readfirstlane(blockIdx.x / a.tiles_n) : 0;
  const uint32_t tile = blockIdx.x - split * a.tiles_n;
  const uint32_t n0 = tile * (16 * RT);
  const uint32_t rows_n = min(uint32_t(a.N) - n0, 16u * RT), M = uint32_t(a.M);

  Walk<RT, TM, DEPTH> walk;
  walk.K = uint32_t(a.K);
  walk.steps = a.steps;
  const uint32_t block = n0 / kF8Group;
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    walk.wq[t] = make_rsrc(a.w[0].codes + int64_t(n0) * a.w[0].ld, (rows_n - 1) * uint32_t(a.w[0].ld) + walk.K);
    walk.ws[t] = make_rsrc(a.w[0].scales + block * a.w[0].lds, a.steps);
    walk.w_off[t] = uint32_t(16 * t + r) * uint32_t(a.w[0].ld);
    if (16u * t + r >= rows_n) walk.w_off[t] = kOutside / 2;
  }
  walk.xq = make_rsrc(a.x, (M - 1) * uint32_t(a.ldx) + walk.K);
  walk.xs = make_rsrc(a.x_scales, (M - 1) * uint32_t(a.ldxs) + a.steps);
#pragma unroll
  for (int u = 0; u < TM; ++u) {
    const uint32_t m = 16 * u + r;
    walk.x_off[u] = m < M ? m * uint32_t(a.ldx) : kOutside / 2;
    walk.xs_off[u] = m < M ? m * uint32_t(a.ldxs) : kOutside / 2;
  }
  f32x4 acc[RT][TM];
#pragma unroll
  for (int t = 0; t < RT; ++t)
#pragma unroll
    for (int u = 0; u < TM; ++u) acc[t][u] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  const uint32_t begin = split * a.steps_per_split, end = min(begin + a.steps_per_split, uint32_t(a.steps));
  walk.run(begin + wave, WAVES, end, acc);

#pragma unroll
  for (int t = 0; t < RT; ++t)
#pragma unroll
    for (int u = 0; u < TM; ++u) *reinterpret_cast<f32x4*>(sums[wave][t * TM + u][lane]) = acc[t][u];
  __syncthreads();
  for (uint32_t part = wave; part < RT * TM; part += WAVES) {
    f32x4 v = *reinterpret_cast<const f32x4*>(sums[0][part][lane]);
#pragma unroll
    for (int i = 1; i < WAVES; ++i) {
      const f32x4 p = *reinterpret_cast<const f32x4*>(sums[i][part][lane]);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += p[e];
    }
    const uint32_t m = part % TM * 16 + r, n = n0 + part / TM * 16 + 4 * g;
    if (m >= M) continue;
    if (a.splits > 1) {  // rows of a multiple of 16 features
      *reinterpret_cast<f32x4*>(a.parts + (int64_t(split) * M + m) * a.ld_parts + n) = v;
      continue;
    }
    using Raw = typename Out::raw;
    Raw* y = static_cast<Raw*>(a.y) + m * a.ldy;
    const Raw* bias = static_cast<const Raw*>(a.bias);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n + e < a.N) y[n + e] = Out::store(bias ? v[e] + Out::load(bias[n + e]) : v[e]);
  }
}

// The splits' parts, added in their order, plus the bias. Four features a thread.
template <class Out>
__global__ void __launch_bounds__(256) join_kernel(const F8JoinArgs a) {
  using Raw = typename Out::raw;
  const uint32_t per_row = uint32_t(a.ld_parts / 4);
  const uint32_t at = blockIdx.x * 256 + threadIdx.x;
  const uint32_t m = at / per_row, n = (at - m * per_row) * 4;
  if (m >= a.M) return;
  const float* p = a.parts + int64_t(m) * a.ld_parts + n;
  const int64_t plane = a.M * a.ld_parts;
  f32x4 v = *reinterpret_cast<const f32x4*>(p);
  for (uint32_t s = 1; s < a.splits; ++s) {
    const f32x4 q = *reinterpret_cast<const f32x4*>(p + s * plane);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] += q[e];
  }
  Raw* y = static_cast<Raw*>(a.y) + m * a.ldy;
  const Raw* bias = static_cast<const Raw*>(a.bias);
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (n + e < a.N) y[n + e] = Out::store(bias ? v[e] + Out::load(bias[n + e]) : v[e]);
}

// silu(x gate^T) * (x up^T), quantized: a workgroup takes a group of 128 features, wave w the 16 from 16 (w % 8) on of gate
// and up, and of the steps every other one.
template <int TM, int DEPTH>
__global__ void __launch_bounds__(1024) decode_gated_kernel(const F8DecodeArgs a) {
  __shared__ __align__(16) float sums[8][2 * TM][64][4];
  __shared__ uint32_t tops[8][16 * TM];
  const int lane = threadIdx.x & 63;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;
  const uint32_t part = wave & 7, half = wave >> 3;
  const uint32_t n0 = blockIdx.x * kF8Group, M = uint32_t(a.M);
  const uint32_t rows_n = min(uint32_t(a.N) - n0, uint32_t(kF8Group));

  Walk<2, TM, DEPTH> walk;
  walk.K = uint32_t(a.K);
  walk.steps = a.steps;
  const uint32_t row = 16 * part + r;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    walk.wq[t] = make_rsrc(a.w[t].codes + int64_t(n0) * a.w[t].ld, (rows_n - 1) * uint32_t(a.w[t].ld) + walk.K);
    walk.ws[t] = make_rsrc(a.w[t].scales + blockIdx.x * a.w[t].lds, a.steps);
    walk.w_off[t] = row < rows_n ? row * uint32_t(a.w[t].ld) : kOutside / 2;
  }
  walk.xq = make_rsrc(a.x, (M - 1) * uint32_t(a.ldx) + walk.K);
  walk.xs = make_rsrc(a.x_scales, (M - 1) * uint32_t(a.ldxs) + a.steps);
#pragma unroll
  for (int u = 0; u < TM; ++u) {
    const uint32_t m = 16 * u + r;
    walk.x_off[u] = m < M ? m * uint32_t(a.ldx) : kOutside / 2;
    walk.xs_off[u] = m < M ? m * uint32_t(a.ldxs) : kOutside / 2;
  }
  f32x4 acc[2][TM];
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int u = 0; u < TM; ++u) acc[t][u] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  walk.run(half, 2, a.steps, acc);

  if (half == 1) {
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int u = 0; u < TM; ++u) *reinterpret_cast<f32x4*>(sums[part][t * TM + u][lane]) = acc[t][u];
  }
  __syncthreads();
  float v[TM][4];
  if (half == 0) {
#pragma unroll
    for (int u = 0; u < TM; ++u) {
      uint32_t top = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float gate = acc[0][u][e] + sums[part][u][lane][e], up = acc[1][u][e] + sums[part][TM + u][lane][e];
        v[u][e] = gate / (1.0f + __expf(-gate)) * up;  // zeros behind the last feature
        top = max(top, magnitude(v[u][e]));
      }
      top = max(top, uint32_t(__shfl_xor(int(top), 16, 64)));
      top = max(top, uint32_t(__shfl_xor(int(top), 32, 64)));
      if (g == 0) tops[part][16 * u + r] = top;
    }
  }
  __syncthreads();
  if (half == 1) return;
#pragma unroll
  for (int u = 0; u < TM; ++u) {
    const uint32_t m = 16 * u + r, n = 16 * part + 4 * g;
    if (m >= M) continue;
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, tops[i][m]);
    const uint32_t scale = f8_scale(top);
    const uint32_t codes = f8_codes4(v[u][0], v[u][1], v[u][2], v[u][3], f8_inverse(scale));
    uint8_t* out = a.codes + int64_t(m) * a.ldc + n0 + n;
    if (a.vec && n + 4 <= rows_n) {
      *reinterpret_cast<uint32_t*>(out) = codes;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n + e < rows_n) out[e] = uint8_t(codes >> (8 * e));
    }
    if (part == 0 && g == 0) a.scales[int64_t(m) * a.lds + blockIdx.x] = uint8_t(scale);
  }
}

template <int RT, int TM, int WAVES, int DEPTH>
hipError_t launch(const F8DecodeArgs& a, int out_dtype, hipStream_t stream) {
  const dim3 grid(a.tiles_n * a.splits), block(64 * WAVES);
  if (out_dtype == kDtF16)
    hipLaunchKernelGGL((decode_kernel<RT, TM, WAVES, DEPTH, ActF16>), grid, block, 0, stream, a);
  else
    hipLaunchKernelGGL((decode_kernel<RT, TM, WAVES, DEPTH, ActBf16>), grid, block, 0, stream, a);
  hipError_t err = hipGetLastError();
  if (err != hipSuccess || a.splits == 1) return err;
  return launch_f8_join({a.parts, a.splits, a.M, a.N, a.ld_parts, a.bias, a.y, a.ldy}, out_dtype, stream);
}

}  // namespace

hipError_t launch_f8_join(const F8JoinArgs& a, int out_dtype, hipStream_t stream) {
  const dim3 grid(uint32_t((a.M * (a.ld_parts / 4) + 255) / 256));
  if (out_dtype == kDtF16)
    hipLaunchKernelGGL(join_kernel<ActF16>, grid, dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL(join_kernel<ActBf16>, grid, dim3(256), 0, stream, a);
  return hipGetLastError();
}

hipError_t launch_f8_decode(const F8DecodeArgs& a, int rt, int out_dtype, hipStream_t stream) {
  const int tm = int((a.M + 15) / 16);
  if (rt == 1) {
    if (tm == 1) return launch<1, 1, 8, 4>(a, out_dtype, stream);
    if (tm == 2) return launch<1, 2, 8, 4>(a, out_dtype, stream);
    return launch<1, 4, 8, 2>(a, out_dtype, stream);
  }
  if (tm == 1) return launch<2, 1, 8, 4>(a, out_dtype, stream);
  if (tm == 2) return launch<2, 2, 8, 2>(a, out_dtype, stream);
  return launch<2, 4, 8, 2>(a, out_dtype, stream);
}

hipError_t launch_f8_decode_gated(const F8DecodeArgs& a, hipStream_t stream) {
  const int tm = int((a.M + 15) / 16);
  const dim3 grid(unsigned((a.N + kF8Group - 1) / kF8Group)), block(1024);
  if (tm == 1)
    hipLaunchKernelGGL((decode_gated_kernel<1, 3>), grid, block, 0, stream, a);
  else if (tm == 2)
    hipLaunchKernelGGL((decode_gated_kernel<2, 2>), grid, block, 0, stream, a);
  else
    hipLaunchKernelGGL((decode_gated_kernel<4, 1>), grid, block, 0, stream, a);
  return hipGetLastError();
}

}  // namespace llmopt
