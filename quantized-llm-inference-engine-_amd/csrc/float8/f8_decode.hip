// The products of up to 16 tokens: bound by the weight's bytes, which go from memory straight into the matrix core's operands.
//
// A workgroup takes 16 features, and its waves the steps of 128 columns in turn, four at a time; their sums are added in LDS
// in a fixed order. What bounds it next to the memory is the rate of a CU's load instructions, 20 ns or so for each that brings a
// kilobyte (25 bytes a cycle; measured): so the tokens' codes come as whole lines (a load of their rows as the matrix core
// wants them would bring each line of one token 16 times) and scales four at a time.
//
// Measured (MI355X, in a graph, weights from memory, us; 1 / 4 / 8 / 16 tokens):
//   6144 x 4096 8.4 / 8.5 / 9.0 / 10.8, 4096 x 14336 13.8 / 13.3 / 14.3 / 16.3 (4.3 TB/s), 28672 x 4096 24.2 / 23.7 / 25.3 / 29.1
//   (4.9 TB/s). With codes and scales loaded by each lane for itself 10.2, 17.5 and 34.3 at one token, 14.7, 19.6 and 43.1 at 16.
//   Four waves a workgroup are up to 12 % faster than eight from 512 workgroups on (28672 x 4096, 16 tokens: 33.0), and as much
//   slower below (4096 x 4096: 7.5 against 7.1); 32 features a workgroup are slower but for 16 tokens at 6144 x 4096 (9.1).
#include "f8_common.hpp"
#include "f8_mfma.hpp"

namespace llmopt {
namespace {

constexpr uint32_t kOutside = 0x7FFFFFF0u;

constexpr uint32_t kGroup = 4;  // steps that a wave takes at a time: four scales are one word

// Sums of 16 weight rows with at most XR tokens over the steps of one wave. The tokens' codes go to LDS of the wave's own,
// the weight's into registers; two groups of steps are on their way.
template <int XR>
struct Walk {
  static constexpr int kXLines = kGroup * XR, kXLoads = (kXLines + 7) / 8;
  static constexpr int kXBytes = kXLoads * 1024;  // of a group
  static constexpr int kLoads = kXLoads + 2 + 2 * int(kGroup);  // (two more for each scale where they are read one by one)

  __amdgpu_buffer_rsrc_t wq, ws, xq, xs;
  uint32_t w_off;  // this lane's row
  uint32_t ldx, xs_off, M, K, steps;
  uint8_t* lds;  // two groups' codes

  struct Slot {
    u32x4 w[kGroup][2];
    uint32_t sw, sx;
  };

  // Four scales from step on, as a word; those behind the end are zeros (a NaN there would reach the sums).
  __device__ __forceinline__ uint32_t scales(__amdgpu_buffer_rsrc_t q, uint32_t off, uint32_t step) const {
    if (step + kGroup <= steps) return __builtin_amdgcn_raw_buffer_load_b32(q, int(off + step), 0, 0);
    uint32_t v = 0;
#pragma unroll
    for (uint32_t i = 0; i < kGroup - 1; ++i)
      v |= uint32_t(__builtin_amdgcn_raw_buffer_load_b8(q, int(step + i < steps ? off + step + i : kOutside), 0, 0)) << (8 * i);
    return v;
  }

  __device__ __forceinline__ void load(Slot& s, uint32_t group, int parity) const {
    const int lane = threadIdx.x & 63, g = lane >> 4;
    const uint32_t step = group * kGroup;
#pragma unroll
    for (int i = 0; i < kXLoads; ++i) {
      const uint32_t line = 8 * i + (lane >> 3), m = line % XR;
      const uint32_t k = (step + line / XR) * kF8Group + 16 * ((lane & 7) ^ (m & 7));
      load_lds16_cached(xq, lds + parity * kXBytes + 1024 * i, line < kXLines && m < M && k < K ? m * ldx + k : kOutside, 0);
    }
    s.sx = scales(xs, xs_off, step);
    s.sw = scales(ws, 0, step);
#pragma unroll
    for (uint32_t j = 0; j < kGroup; ++j) {
      const uint32_t k = (step + j) * kF8Group + 16 * g;
      s.w[j][0] = buf_load16(wq, k < K ? w_off + k : kOutside, 0);
      s.w[j][1] = buf_load16(wq, k + 64 < K ? w_off + k + 64 : kOutside, 0);
    }
  }

  __device__ __forceinline__ void multiply(const Slot& s, int parity, f32x4& acc) const {
    const int lane = threadIdx.x & 63, g = lane >> 4, m = (lane & 15) % XR;
    auto one = [&](auto step) {
      constexpr int J = decltype(step)::value;
      const uint8_t* at = lds + parity * kXBytes + (J * XR + m) * kF8Group;
      const u32x4 lo = *reinterpret_cast<const u32x4*>(at + 16 * (g ^ (m & 7)));
      const u32x4 hi = *reinterpret_cast<const u32x4*>(at + 16 * ((g + 4) ^ (m & 7)));
      const i32x8 x = __builtin_bit_cast(i32x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
      const i32x8 w = __builtin_bit_cast(i32x8, __builtin_shufflevector(s.w[J][0], s.w[J][1], 0, 1, 2, 3, 4, 5, 6, 7));
      acc = mfma_f8<J, J>(w, x, acc, s.sw, s.sx);
    };
    one(std::integral_constant<int, 0>{});
    one(std::integral_constant<int, 1>{});
    one(std::integral_constant<int, 2>{});
    one(std::integral_constant<int, 3>{});
  }

  // Groups first, first + stride, ... below end.
  __device__ __forceinline__ void run(uint32_t first, uint32_t stride, uint32_t end, f32x4& acc) const {
    if (first >= end) return;
    Slot slot[2];
    load(slot[0], first, 0);
    auto turn = [&](uint32_t group, auto parity) {
      constexpr int P = decltype(parity)::value;
      __builtin_amdgcn_sched_barrier(0);
      if (group + stride < end) {
        load(slot[1 - P], group + stride, 1 - P);
        __builtin_amdgcn_sched_barrier(0);
        wait_vmcnt<kLoads>();  // all but those of the next group
      } else {
        wait_vmcnt<0>();
      }
      __builtin_amdgcn_sched_barrier(0);
      multiply(slot[P], P, acc);
      wait_lgkmcnt0();  // before its LDS is loaded anew
    };
    for (uint32_t group = first; group < end; group += 2 * stride) {
      turn(group, std::integral_constant<int, 0>{});
      if (group + stride < end) turn(group + stride, std::integral_constant<int, 1>{});
    }
  }
};

// y of 16 features and M <= XR tokens. With a second weight the workgroups behind `tiles` take that one, and their rows of y come
// behind the first one's.
template <int XR, int WAVES, class Out>
__global__ void __launch_bounds__(64 * WAVES) decode_kernel(const F8DecodeArgs a) {
  using W = Walk<XR>;
  __shared__ __align__(1024) uint8_t codes[WAVES][2 * W::kXBytes];
  __shared__ __align__(16) float sums[WAVES][64][4];
  const int lane = threadIdx.x & 63;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t r = lane & 15, g = lane >> 4;
  const bool second = blockIdx.x >= a.tiles;
  const F8Weight w = second ? a.w[1] : a.w[0];
  const uint32_t n0 = (second ? blockIdx.x - a.tiles : blockIdx.x) * 16;
  const uint32_t rows_n = min(uint32_t(a.N) - n0, 16u), M = uint32_t(a.M);

  W walk;
  walk.K = uint32_t(a.K);
  walk.M = M;
  walk.steps = a.steps;
  walk.ldx = uint32_t(a.ldx);
  walk.xq = make_rsrc(a.x, (M - 1) * walk.ldx + walk.K);
  walk.xs = make_rsrc(a.x_scales, (M - 1) * uint32_t(a.ldxs) + a.steps);
  walk.xs_off = min(r, M - 1) * uint32_t(a.ldxs);
  walk.lds = codes[wave];
  walk.wq = make_rsrc(w.codes + int64_t(n0) * w.ld, (rows_n - 1) * uint32_t(w.ld) + walk.K);
  walk.ws = make_rsrc(w.scales + n0 / kF8Group * w.lds, a.steps);
  walk.w_off = r < rows_n ? r * uint32_t(w.ld) : kOutside / 2;  // rows behind the last read as zeros
  f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
  walk.run(wave, WAVES, (a.steps + kGroup - 1) / kGroup, acc);

  *reinterpret_cast<f32x4*>(sums[wave][lane]) = acc;
  __syncthreads();
  if (wave != 0 || r >= M) return;
#pragma unroll
  for (int i = 1; i < WAVES; ++i) {
    const f32x4 p = *reinterpret_cast<const f32x4*>(sums[i][lane]);
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] += p[e];
  }
  const uint32_t n = n0 + 4 * g;
  using Raw = typename Out::raw;
  Raw* y = static_cast<Raw*>(a.y) + (second ? M + r : r) * a.ldy;
  const Raw* bias = static_cast<const Raw*>(a.bias);
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (n + e < a.N) y[n + e] = Out::store(bias ? acc[e] + Out::load(bias[n + e]) : acc[e]);
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

template <int XR, int WAVES>
hipError_t launch(const F8DecodeArgs& a, int out_dtype, hipStream_t stream) {
  const dim3 grid(a.tiles * (a.w[1].codes ? 2 : 1)), block(64 * WAVES);
  if (out_dtype == kDtF32)
    hipLaunchKernelGGL((decode_kernel<XR, WAVES, ActF32>), grid, block, 0, stream, a);
  else if (out_dtype == kDtF16)
    hipLaunchKernelGGL((decode_kernel<XR, WAVES, ActF16>), grid, block, 0, stream, a);
  else
    hipLaunchKernelGGL((decode_kernel<XR, WAVES, ActBf16>), grid, block, 0, stream, a);
  return hipGetLastError();
}

template <int WAVES>
hipError_t launch_rows(const F8DecodeArgs& a, int out_dtype, hipStream_t stream) {
  if (a.M == 1) return launch<1, WAVES>(a, out_dtype, stream);
  if (a.M <= 4) return launch<4, WAVES>(a, out_dtype, stream);
  if (a.M <= 8) return launch<8, WAVES>(a, out_dtype, stream);
  return launch<16, WAVES>(a, out_dtype, stream);
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

hipError_t launch_f8_decode(F8DecodeArgs a, int out_dtype, hipStream_t stream) {
  a.steps = uint32_t((a.K + kF8Group - 1) / kF8Group);
  a.tiles = uint32_t((a.N + 15) / 16);
  const uint32_t count = a.tiles * (a.w[1].codes ? 2 : 1);
  return count >= 512 ? launch_rows<4>(a, out_dtype, stream) : launch_rows<8>(a, out_dtype, stream);
}

}  // namespace llmopt
