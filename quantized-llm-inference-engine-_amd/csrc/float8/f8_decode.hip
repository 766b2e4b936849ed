// The products of few tokens, up to 16 of any weight and more where llmopt_f8_linear's estimate says so: bound by the weight's bytes.
//
// A workgroup takes 16 features, and its waves the steps of 128 columns in turn, four at a time; their sums are added in LDS
// in a fixed order. What bounds it next to the memory is a CU's load instructions: one of eight whole lines takes it 8 ns, one
// of 16 half lines 15 (measured on cached data). So codes come as whole lines straight into LDS of the wave's own (loaded into the
// matrix core's operands, a line of one token would be asked for 16 times), and scales four at a time.
//
// Measured (MI355X, in a graph, weights from memory, us; 1 / 4 / 8 / 16 tokens):
//   6144 x 4096 7.2 / 7.4 / 9.1 / 10.0, 4096 x 14336 11.6 / 11.9 / 12.0 / 13.0 (5.0 TB/s), 28672 x 4096 22.3 / 22.7 / 26.1 / 28.9
//   (5.3 TB/s), 1536 x 1024 2.9 / 3.0 / 3.1 / 3.1.
// Codes and scales loaded by each lane for itself: 10.2, 17.5 and 34.3 at one token, 14.7, 19.6 and 43.1 at 16.
// The weight's codes into registers (HELD) instead of LDS: 8.4, 13.7, 24.2 and 3.3 at one token, but at more than four tokens, whose
// LDS leaves room for fewer waves, faster from some 640 workgroups on where a row has more than 16 steps, for eight waves (in LDS /
// HELD, 8 and 16 tokens: 28672 x 4096 29.5 / 27.6 and 32.2 / 29.4, 16384 x 4096 18.3 / 17.1 and 19.6 / 18.6, 10240 x 4096 the
// same; with 16 steps, for four waves: 28672 x 2048 13.6 / 14.7 and 15.8 / 16.2, 10240 x 2048 6.7 / 7.5 and 7.5 / 8.2, with eight
// waves, half of which have none, 16.5 and 17.8, 8.2 and 8.4; 28672 x 1024 9.3 / 9.7 and 10.9 / 10.8).
// More than 16 tokens go 32 at a time: their codes fill LDS with one workgroup a CU (two where a row has at most 16 steps), and the
// weight's are HELD. 32 / 64 / 100 tokens, in brackets the best of the tiles: 1536 x 1024 3.9 / 3.9 / 4.5 (8.3), 4096 x 4096 8.6 (13.0) / 13.2 (13.2) / -,
// 1024 x 2816 5.8 / 5.8 / 5.9 (9.4 - 10), 6144 x 4096 13.3 (14.0), 4096 x 14336 19.5 (18.6), 28672 x 4096 40 (30).
// Eight waves where each has one group of steps (17 to 32 steps; no second buffer), else four: 4096 x 4096 5.6 against 5.7 (16
// tokens 6.6 against 6.8), 4096 x 14336 11.7 against 11.6 (4 tokens 12.2 against 11.9), 1024 x 2816 4.1 against 3.9, 8192 x 2048 at 16
// tokens 7.3 against 5.6.
#include "f8_common.hpp"
#include "f8_mfma.hpp"

namespace llmopt {
namespace {

constexpr uint32_t kOutside = 0x7FFFFFF0u;

constexpr uint32_t kGroup = 4;  // steps that a wave takes at a time: four scales are one word

// Sums of 16 weight rows with at most XR tokens over the steps of one wave. The tokens' codes go to LDS of the wave's own, the
// weight's too (whole lines, past the caches) or into registers (HELD); up to two groups of steps are on their way.
template <int XR, bool HELD>
struct Walk {
  static constexpr int kXLines = kGroup * XR, kXLoads = (kXLines + 7) / 8;
  static constexpr int kWLoads = 2 * int(kGroup);
  static constexpr int kTiles = XR > 16 ? XR / 16 : 1;  // of 16 tokens
  static constexpr int kWBytes = HELD ? 0 : kWLoads * 1024, kBytes = kWBytes + kXLoads * 1024;  // of a group, in LDS
  static constexpr int kLoads = kXLoads + kTiles + 1 + kWLoads;  // (two more for each scale where they are read one by one)

  __amdgpu_buffer_rsrc_t wq, ws, xq, xs;
  uint32_t w_off[2];  // HELD: this lane's row; else the two that it brings
  uint32_t xs_off[kTiles], ldx, M, K, steps;
  uint8_t* lds;

  struct Slot {
    u32x4 w[HELD ? kGroup : 1][2];
    uint32_t sw, sx[kTiles];
  };

  // Of weight rows from n0 on and the M <= XR tokens from m0 on.
  __device__ __forceinline__ Walk(const F8DecodeArgs& a, const F8Weight& w, uint32_t n0, uint32_t m0, uint8_t* lds_) {
    const uint32_t lane = threadIdx.x & 63, r = lane & 15, rows = min(uint32_t(a.N) - n0, 16u);
    K = uint32_t(a.K);
    M = XR == 1 ? 1 : XR > 16 ? min(uint32_t(a.M) - m0, uint32_t(XR)) : uint32_t(a.M);
    steps = a.steps;
    ldx = uint32_t(a.ldx);
    lds = lds_;
    xq = make_rsrc(a.x + int64_t(m0) * a.ldx, (M - 1) * ldx + K);
    xs = make_rsrc(a.x_scales + int64_t(m0) * a.ldxs, (M - 1) * uint32_t(a.ldxs) + steps);
#pragma unroll
    for (int t = 0; t < kTiles; ++t) xs_off[t] = min(16 * t + r, M - 1) * uint32_t(a.ldxs);
    wq = make_rsrc(w.codes + int64_t(n0) * w.ld, (rows - 1) * uint32_t(w.ld) + K);
    ws = make_rsrc(w.scales + n0 / kF8Group * w.lds, steps);
#pragma unroll
    for (uint32_t h = 0; h < 2; ++h) {
      const uint32_t row = HELD ? r : 8 * h + (lane >> 3);
      w_off[h] = row < rows ? row * uint32_t(w.ld) : kOutside / 2;  // rows behind the last read as zeros
    }
  }

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
    const uint32_t lane = threadIdx.x & 63, step = group * kGroup;
    uint8_t* const to = lds + parity * kBytes;
#pragma unroll
    for (int i = 0; i < kXLoads; ++i) {
      const uint32_t line = 8 * i + (lane >> 3), m = line % XR;
      const uint32_t k = (step + line / XR) * kF8Group + 16 * ((lane & 7) ^ (m & 7));
      load_lds16_cached(xq, to + kWBytes + 1024 * i, line < kXLines && m < M && k < K ? m * ldx + k : kOutside, 0);
    }
#pragma unroll
    for (int t = 0; t < kTiles; ++t) s.sx[t] = scales(xs, xs_off[t], step);
    s.sw = scales(ws, 0, step);
#pragma unroll
    for (int i = 0; i < kWLoads; ++i) {
      if constexpr (HELD) {  // half the columns of a step for each row
        const uint32_t k = (step + i / 2) * kF8Group + 64 * (i & 1) + 16 * (lane >> 4);
        s.w[i / 2][i & 1] = buf_load16(wq, k < K ? w_off[0] + k : kOutside, 0);
      } else {  // a step for eight rows
        const uint32_t k = (step + i / 2) * kF8Group + 16 * ((lane & 7) ^ (lane >> 3));
        load_lds16(wq, to + 1024 * i, k < K ? w_off[i & 1] + k : kOutside, 0);
      }
    }
  }

  __device__ __forceinline__ void multiply(const Slot& s, int parity, f32x4 (&acc)[kTiles]) const {
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const uint8_t* const from = lds + parity * kBytes;
    auto operand = [&](const uint8_t* line, int swizzle) {
      const u32x4 lo = *reinterpret_cast<const u32x4*>(line + 16 * (g ^ swizzle));
      const u32x4 hi = *reinterpret_cast<const u32x4*>(line + 16 * ((g + 4) ^ swizzle));
      return __builtin_bit_cast(i32x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    };
    auto one = [&](auto step) {
      constexpr int J = decltype(step)::value;
      i32x8 w;
      if constexpr (HELD)
        w = __builtin_bit_cast(i32x8, __builtin_shufflevector(s.w[J][0], s.w[J][1], 0, 1, 2, 3, 4, 5, 6, 7));
      else
        w = operand(from + (J * 16 + r) * kF8Group, r & 7);
#pragma unroll
      for (int t = 0; t < kTiles; ++t) {
        const int m = 16 * t + r % XR;
        acc[t] = mfma_f8<J, J>(w, operand(from + kWBytes + (J * XR + m) * kF8Group, m & 7), acc[t], s.sw, s.sx[t]);
      }
    };
    one(std::integral_constant<int, 0>{});
    one(std::integral_constant<int, 1>{});
    one(std::integral_constant<int, 2>{});
    one(std::integral_constant<int, 3>{});
  }

  // Groups first, first + stride, ... below end.
  __device__ __forceinline__ void run(uint32_t first, uint32_t stride, uint32_t end, f32x4 (&acc)[kTiles]) const {
    if (first >= end) return;
    Slot slot[2];
    load(slot[0], first, 0);
    auto turn = [&](uint32_t group, auto parity) {
      constexpr int P = decltype(parity)::value;
      __builtin_amdgcn_sched_barrier(0);
      if (group + stride < end) {
        load(slot[1 - P], group + stride, 1 - P);
        __builtin_amdgcn_sched_barrier(0);
        wait_vmcnt<kLoads>();  // all but those of the next group, which are as many at least
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

// y of 16 features and at most XR tokens (blockIdx.y counts them). With a second weight the workgroups behind `tiles` take that one, and their rows of y come
// behind the first one's. LDS: `buffers` groups of each wave (two where a wave has more than one).
template <int XR, bool HELD, int WAVES, class Out>
__global__ void __launch_bounds__(64 * WAVES) decode_kernel(const F8DecodeArgs a, int buffers) {
  using W = Walk<XR, HELD>;
  static_assert(W::kBytes >= 1024 * W::kTiles, "room for a wave's sums");
  extern __shared__ __align__(1024) uint8_t lds[];
  const int lane = threadIdx.x & 63;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t r = lane & 15, g = lane >> 4, m0 = XR > 16 ? blockIdx.y * XR : 0;
  const bool second = blockIdx.x >= a.tiles;
  const uint32_t n0 = (second ? blockIdx.x - a.tiles : blockIdx.x) * 16;
  uint8_t* const own = lds + wave * uint32_t(buffers * W::kBytes);

  const W walk(a, second ? a.w[1] : a.w[0], n0, m0, own);
  f32x4 acc[W::kTiles];
#pragma unroll
  for (int t = 0; t < W::kTiles; ++t) acc[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  walk.run(wave, WAVES, (a.steps + kGroup - 1) / kGroup, acc);

  // (nothing is on its way there any more)
#pragma unroll
  for (int t = 0; t < W::kTiles; ++t) *reinterpret_cast<f32x4*>(own + 1024 * t + 16 * lane) = acc[t];
  __syncthreads();
  const int64_t m = m0 + 16 * wave + r;  // a wave for each 16 tokens
  if (wave >= W::kTiles || (XR < 16 && r >= XR) || m >= a.M) return;
  f32x4 sum = acc[0];  // of one tile wave 0 has the first summand
  if constexpr (W::kTiles > 1) sum = *reinterpret_cast<const f32x4*>(lds + 1024 * wave + 16 * lane);
#pragma unroll
  for (int i = 1; i < WAVES; ++i) {
    const f32x4 p = *reinterpret_cast<const f32x4*>(lds + i * buffers * W::kBytes + 1024 * wave + 16 * lane);
#pragma unroll
    for (int e = 0; e < 4; ++e) sum[e] += p[e];
  }
  const uint32_t n = n0 + 4 * g;
  using Raw = typename Out::raw;
  Raw* y = static_cast<Raw*>(a.y) + (second ? a.M + m : m) * a.ldy;
  const Raw* bias = static_cast<const Raw*>(a.bias);
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (n + e < a.N) y[n + e] = Out::store(bias ? sum[e] + Out::load(bias[n + e]) : sum[e]);
}

// The splits' parts, added in their order, plus the bias. Four features a thread, all their parts on their way at once.
template <int SPLITS, class Out>
__global__ void __launch_bounds__(256) join_kernel(const F8JoinArgs a) {
  using Raw = typename Out::raw;
  const uint32_t per_row = uint32_t(a.ld_parts / 4);
  const uint32_t at = blockIdx.x * 256 + threadIdx.x;
  const uint32_t m = at / per_row, n = (at - m * per_row) * 4;
  if (m >= a.M) return;
  const float* p = a.parts + int64_t(m) * a.ld_parts + n;
  const int64_t plane = a.M * a.ld_parts;
  f32x4 part[SPLITS];
#pragma unroll
  for (int s = 0; s < SPLITS; ++s) part[s] = *reinterpret_cast<const f32x4*>(p + s * plane);
  f32x4 v = part[0];
#pragma unroll
  for (int s = 1; s < SPLITS; ++s)
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] += part[s][e];
  Raw* y = static_cast<Raw*>(a.y) + m * a.ldy;
  const Raw* bias = static_cast<const Raw*>(a.bias);
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (n + e < a.N) y[n + e] = Out::store(bias ? v[e] + Out::load(bias[n + e]) : v[e]);
}

template <class Out>
hipError_t launch_join(const F8JoinArgs& a, hipStream_t stream) {
  const dim3 grid(uint32_t((a.M * (a.ld_parts / 4) + 255) / 256));
  switch (a.splits) {
    case 2: hipLaunchKernelGGL((join_kernel<2, Out>), grid, dim3(256), 0, stream, a); break;
    case 4: hipLaunchKernelGGL((join_kernel<4, Out>), grid, dim3(256), 0, stream, a); break;
    case 8: hipLaunchKernelGGL((join_kernel<8, Out>), grid, dim3(256), 0, stream, a); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

template <int XR, bool HELD, int WAVES, class Out>
hipError_t launch_out(const F8DecodeArgs& a, hipStream_t stream) {
  auto* kernel = decode_kernel<XR, HELD, WAVES, Out>;
  const int buffers = a.steps > kGroup * WAVES ? 2 : 1, bytes = WAVES * buffers * Walk<XR, HELD>::kBytes;
  if (bytes > 64 * 1024) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL(kernel, dim3(a.tiles * (a.w[1].codes ? 2 : 1), uint32_t((a.M + XR - 1) / XR)), dim3(64 * WAVES), bytes, stream, a, buffers);
  return hipGetLastError();
}

template <int XR, bool HELD, int WAVES>
hipError_t launch(const F8DecodeArgs& a, int out_dtype, hipStream_t stream) {
  if (out_dtype == kDtF32) return launch_out<XR, HELD, WAVES, ActF32>(a, stream);
  if (out_dtype == kDtF16) return launch_out<XR, HELD, WAVES, ActF16>(a, stream);
  return launch_out<XR, HELD, WAVES, ActBf16>(a, stream);
}

template <int XR>
hipError_t launch_rows(const F8DecodeArgs& a, int out_dtype, hipStream_t stream) {
  const bool one_group = a.steps > 16 && a.steps <= 32;  // of each of eight waves
  if constexpr (XR > 16) {
    return one_group ? launch<XR, true, 8>(a, out_dtype, stream) : launch<XR, true, 4>(a, out_dtype, stream);
  } else {
    if constexpr (XR > 4) {
      if (a.steps > 16 && a.tiles * (a.w[1].codes ? 2 : 1) >= 640) return launch<XR, true, 8>(a, out_dtype, stream);
    }
    return one_group ? launch<XR, false, 8>(a, out_dtype, stream) : launch<XR, false, 4>(a, out_dtype, stream);
  }
}

}  // namespace

hipError_t launch_f8_join(const F8JoinArgs& a, int out_dtype, hipStream_t stream) {
  return out_dtype == kDtF16 ? launch_join<ActF16>(a, stream) : launch_join<ActBf16>(a, stream);
}

hipError_t launch_f8_decode(F8DecodeArgs a, int out_dtype, hipStream_t stream) {
  a.steps = uint32_t((a.K + kF8Group - 1) / kF8Group);
  a.tiles = uint32_t((a.N + 15) / 16);
  if (a.M == 1) return launch_rows<1>(a, out_dtype, stream);
  if (a.M <= 4) return launch_rows<4>(a, out_dtype, stream);
  if (a.M <= 8) return launch_rows<8>(a, out_dtype, stream);
  if (a.M <= 16) return launch_rows<16>(a, out_dtype, stream);
  return launch_rows<32>(a, out_dtype, stream);
}

}  // namespace llmopt
