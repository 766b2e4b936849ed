// Quantizing rows and weights into 8-bit floating point, RMSNorm with the residual's addition and a quantized output, and
// the gated activation's quantizing (llmopt_float8.h).
//
// One pass over the data, bound by its bytes: eight numbers a thread, a group's largest magnitude over 16 lanes by DPP (or a whole
// 128 x 128 block held in a workgroup's registers), the scale from its exponent, codes by the hardware's conversion. A scale
// is a power of two, so x / 2^e is exact and the only rounding is the conversion's, half a step of e4m3.
//
// Measured (MI355X, us; floor: the bytes at a large copy's 5.14 TB/s): a weight of 4096 x 14336 bf16 37.3 (34.3); residual and norm of
// 8192 tokens of 4096 49.9 (45.7; with rows read a second time instead of held 53.0); rows quantized, in a graph, 8192 of 4096 21.3
// (19.6), 8192 of 1024 8.5 (4.9), 2048 of 4096 7.2 (4.9), 777 of 1024 2.7 (0.5); from Python 777 tokens of 1024 normed 5.5, one token of 4096
// quantized 4.9 - 5.4 and normed 5.9, of which the kernels take 3.4, 1.8 and 3.5 and the call from Python the rest. Codes are
// stored past the caches (a weight 39.6 us through them).
#include "f8_common.hpp"

namespace llmopt {
namespace {

constexpr int kThreads = 256;
constexpr int kChunk = 8 * kThreads;  // columns of a workgroup

// A workgroup takes `kChunk` columns of a row.
template <class Act>
__global__ void __launch_bounds__(kThreads) quantize_rows_kernel(const F8QuantArgs a, uint32_t chunks) {
  const int64_t row = blockIdx.x / chunks;
  const int64_t c = int64_t(blockIdx.x - uint32_t(row) * chunks) * kChunk + 8 * threadIdx.x;
  float v[8];
  load8<Act>(static_cast<const typename Act::raw*>(a.x) + row * a.ldx, c, a.cols, a.vec, v);
  quantize8(v, a.codes + row * a.ldc, a.scales + row * a.lds, c, a.cols, a.vec);
}

// A workgroup takes a block of 128 x 128: thread t the columns 8 (t % 16) .. of the rows t / 16 + 16 i.
template <class Act>
__global__ void __launch_bounds__(kThreads) quantize_blocks_kernel(const F8QuantArgs a, uint32_t across) {
  __shared__ uint32_t part[kThreads / 64];
  const uint32_t up = blockIdx.x / across, at = blockIdx.x - up * across;
  const int tid = threadIdx.x;
  const int64_t c = int64_t(at) * kF8Group + 8 * (tid & 15);
  float v[8][8];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t r = int64_t(up) * kF8Group + (tid >> 4) + 16 * i;
    const bool in = r < a.rows;
    load8<Act>(static_cast<const typename Act::raw*>(a.x) + (in ? r : 0) * a.ldx, c, in ? a.cols : 0, a.vec, v[i]);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) top = max(top, magnitude(v[i][e]));
  top = max16(top);
  top = max(top, uint32_t(__shfl_xor(int(top), 16, 64)));
  top = max(top, uint32_t(__shfl_xor(int(top), 32, 64)));
  if ((tid & 63) == 0) part[tid >> 6] = top;
  __syncthreads();
  const uint32_t s = f8_scale(max(max(part[0], part[1]), max(part[2], part[3])));
  const float inv = f8_inverse(s);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int64_t r = int64_t(up) * kF8Group + (tid >> 4) + 16 * i;
    const u32x2 w = {f8_codes4(v[i][0], v[i][1], v[i][2], v[i][3], inv), f8_codes4(v[i][4], v[i][5], v[i][6], v[i][7], inv)};
    if (r < a.rows) store_codes8(a.codes + r * a.ldc, c, a.cols, a.vec, w);
  }
  if (tid == 0) a.scales[up * a.lds + at] = uint8_t(s);
}

// h = residual + x rounded to the type, or x, of the eight columns from c on.
template <class Act>
__device__ __forceinline__ void stream8(const F8NormArgs& a, int64_t row, int64_t c, float* h) {
  using Raw = typename Act::raw;
  load8<Act>(static_cast<const Raw*>(a.x) + row * a.ldx, c, a.hidden, a.vec, h);
  if (a.residual) {
    float r[8];
    load8<Act>(static_cast<const Raw*>(a.residual) + row * a.ldr, c, a.hidden, a.vec, r);
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = Act::load(Act::store(r[i] + h[i]));
  }
}

template <class Act>
__device__ __forceinline__ void store_stream8(const F8NormArgs& a, int64_t row, int64_t c, const float* h) {
  using Raw = typename Act::raw;
  Raw* out = static_cast<Raw*>(a.h_out) + row * a.ldh;
  if (a.vec) {
    if (c >= a.hidden) return;
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = uint32_t(Act::store(h[2 * i])) | (uint32_t(Act::store(h[2 * i + 1])) << 16);
    *reinterpret_cast<u32x4*>(out + c) = w;
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (c + i < a.hidden) out[c + i] = Act::store(h[i]);
}

// A workgroup per row of any length; the stream is read again for the second pass (from h_out, which may be x or the
// residual: each thread reads there what it wrote itself).
template <class Act>
__global__ void __launch_bounds__(kThreads) rmsnorm_rows_kernel(const F8NormArgs a) {
  using Raw = typename Act::raw;
  __shared__ float part[kThreads / 64];
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x;
  float ss = 0.0f;
  for (int64_t c = 8 * tid; c < a.hidden; c += kChunk) {
    float h[8];
    stream8<Act>(a, row, c, h);
    if (a.residual) store_stream8<Act>(a, row, c, h);
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = __builtin_fmaf(h[i], h[i], ss);
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) ss += __shfl_xor(ss, off, 64);
  if ((tid & 63) == 0) part[tid >> 6] = ss;
  __syncthreads();
  const float total = (part[0] + part[1]) + (part[2] + part[3]);
  const float inv = __frsqrt_rn(total / float(a.hidden) + a.eps);
  const Raw* src = a.residual ? static_cast<const Raw*>(a.h_out) + row * a.ldh : static_cast<const Raw*>(a.x) + row * a.ldx;
  for (int64_t base = 0; base < a.hidden; base += kChunk) {
    const int64_t c = base + 8 * tid;
    float h[8], w[8];
    load8<Act>(src, c, a.hidden, a.vec, h);
    load8<Act>(static_cast<const Raw*>(a.weight), c, a.hidden, a.vec, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = h[i] * inv * w[i];
    quantize8(h, a.codes + row * a.ldc, a.scales + row * a.lds, c, a.hidden, a.vec);
  }
}

// Rows of up to kThreads * 8 * NIT: the stream stays in registers between the two passes, and everything that is read is on
// its way at once.
template <class Act, int NIT>
__global__ void __launch_bounds__(kThreads) rmsnorm_held_kernel(const F8NormArgs a) {
  using Raw = typename Act::raw;
  __shared__ float part[kThreads / 64];
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x;
  float h[NIT][8], w[NIT][8];
#pragma unroll
  for (int i = 0; i < NIT; ++i) stream8<Act>(a, row, 8 * tid + i * kChunk, h[i]);
#pragma unroll
  for (int i = 0; i < NIT; ++i) load8<Act>(static_cast<const Raw*>(a.weight), 8 * tid + i * kChunk, a.hidden, a.vec, w[i]);
  float ss = 0.0f;
#pragma unroll
  for (int i = 0; i < NIT; ++i) {
    if (a.residual) store_stream8<Act>(a, row, 8 * tid + i * kChunk, h[i]);
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = __builtin_fmaf(h[i][e], h[i][e], ss);
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) ss += __shfl_xor(ss, off, 64);
  if ((tid & 63) == 0) part[tid >> 6] = ss;
  __syncthreads();
  const float total = (part[0] + part[1]) + (part[2] + part[3]);
  const float inv = __frsqrt_rn(total / float(a.hidden) + a.eps);
#pragma unroll
  for (int i = 0; i < NIT; ++i) {
#pragma unroll
    for (int e = 0; e < 8; ++e) h[i][e] = h[i][e] * inv * w[i][e];
    quantize8(h[i], a.codes + row * a.ldc, a.scales + row * a.lds, 8 * tid + i * kChunk, a.hidden, a.vec);
  }
}

// silu(gate) * up, a workgroup per `kChunk` columns of a row.
__global__ void __launch_bounds__(kThreads) act_kernel(const F8ActArgs a, uint32_t chunks, int vec) {
  const int64_t row = blockIdx.x / chunks;
  const int64_t c = int64_t(blockIdx.x - uint32_t(row) * chunks) * kChunk + 8 * threadIdx.x;
  float g[1][8], u[8];
  load8<ActF32>(a.gate + row * a.ld, c, a.cols, vec, g[0]);
  load8<ActF32>(a.up + row * a.ld, c, a.cols, vec, u);
#pragma unroll
  for (int i = 0; i < 8; ++i) g[0][i] = f8_swiglu(g[0][i], u[i]);
  uint32_t top[1] = {largest8(g[0])};
  f8_settle<false, 48>([&] { return a.in; }, g, top, row, c);
  quantize8(g[0], top[0], a.codes + row * a.ldc, a.scales + row * a.lds, c, a.cols, vec);
}

}  // namespace

// Work-items of a launch are counted in 32 bits.
constexpr int64_t kMostGroups = (int64_t(1) << 32) / kThreads - 1;

hipError_t launch_f8_quantize(const F8QuantArgs& a, int dtype, int64_t block_rows, hipStream_t stream) {
  if (a.rows == 0 || a.cols == 0) return hipSuccess;
  if (block_rows == 1) {
    const int64_t chunks = (a.cols + kChunk - 1) / kChunk, most = kMostGroups / chunks;
    if (a.rows > most) {  // in two calls
      F8QuantArgs part = a;
      part.rows = most;
      const hipError_t err = launch_f8_quantize(part, dtype, 1, stream);
      if (err != hipSuccess) return err;
      part.x = static_cast<const uint8_t*>(a.x) + most * a.ldx * (dtype == kDtF32 ? 4 : 2);
      part.codes += most * a.ldc;
      part.scales += most * a.lds;
      part.rows = a.rows - most;
      return launch_f8_quantize(part, dtype, 1, stream);
    }
    const dim3 grid(unsigned(a.rows * chunks));
    if (dtype == kDtF32)
      hipLaunchKernelGGL(quantize_rows_kernel<ActF32>, grid, dim3(kThreads), 0, stream, a, uint32_t(chunks));
    else if (dtype == kDtF16)
      hipLaunchKernelGGL(quantize_rows_kernel<ActF16>, grid, dim3(kThreads), 0, stream, a, uint32_t(chunks));
    else
      hipLaunchKernelGGL(quantize_rows_kernel<ActBf16>, grid, dim3(kThreads), 0, stream, a, uint32_t(chunks));
    return hipGetLastError();
  }
  const int64_t across = (a.cols + kF8Group - 1) / kF8Group;
  const dim3 grid(unsigned(across * ((a.rows + kF8Group - 1) / kF8Group)));
  if (dtype == kDtF32)
    hipLaunchKernelGGL(quantize_blocks_kernel<ActF32>, grid, dim3(kThreads), 0, stream, a, uint32_t(across));
  else if (dtype == kDtF16)
    hipLaunchKernelGGL(quantize_blocks_kernel<ActF16>, grid, dim3(kThreads), 0, stream, a, uint32_t(across));
  else
    hipLaunchKernelGGL(quantize_blocks_kernel<ActBf16>, grid, dim3(kThreads), 0, stream, a, uint32_t(across));
  return hipGetLastError();
}

template <class Act>
static hipError_t launch_norm(const F8NormArgs& a, hipStream_t stream) {
  const dim3 grid(unsigned(a.rows)), block(kThreads);
  if (a.hidden <= kChunk)
    hipLaunchKernelGGL((rmsnorm_held_kernel<Act, 1>), grid, block, 0, stream, a);
  else if (a.hidden <= 2 * kChunk)
    hipLaunchKernelGGL((rmsnorm_held_kernel<Act, 2>), grid, block, 0, stream, a);
  else if (a.hidden <= 4 * kChunk)
    hipLaunchKernelGGL((rmsnorm_held_kernel<Act, 4>), grid, block, 0, stream, a);
  else
    hipLaunchKernelGGL(rmsnorm_rows_kernel<Act>, grid, block, 0, stream, a);
  return hipGetLastError();
}

hipError_t launch_f8_rmsnorm(const F8NormArgs& a, int dtype, hipStream_t stream) {
  if (a.rows == 0 || a.hidden == 0) return hipSuccess;
  if (a.rows > kMostGroups) {  // in two calls
    F8NormArgs part = a;
    part.rows = kMostGroups;
    const hipError_t err = launch_f8_rmsnorm(part, dtype, stream);
    if (err != hipSuccess) return err;
    part.x = static_cast<const uint16_t*>(a.x) + kMostGroups * a.ldx;
    if (a.residual) {
      part.residual = static_cast<const uint16_t*>(a.residual) + kMostGroups * a.ldr;
      part.h_out = static_cast<uint16_t*>(a.h_out) + kMostGroups * a.ldh;
    }
    part.codes += kMostGroups * a.ldc;
    part.scales += kMostGroups * a.lds;
    part.rows = a.rows - kMostGroups;
    return launch_f8_rmsnorm(part, dtype, stream);
  }
  return dtype == kDtF16 ? launch_norm<ActF16>(a, stream) : launch_norm<ActBf16>(a, stream);
}

hipError_t launch_f8_act(const F8ActArgs& a, hipStream_t stream) {
  if (a.rows == 0 || a.cols == 0) return hipSuccess;
  const int64_t chunks = (a.cols + kChunk - 1) / kChunk;
  const int vec = a.cols % 8 == 0 && a.ld % 4 == 0 && a.ldc % 8 == 0 && reinterpret_cast<uintptr_t>(a.gate) % 16 == 0 &&
                  reinterpret_cast<uintptr_t>(a.up) % 16 == 0 && reinterpret_cast<uintptr_t>(a.codes) % 8 == 0;
  hipLaunchKernelGGL(act_kernel, dim3(unsigned(a.rows * chunks)), dim3(kThreads), 0, stream, a, uint32_t(chunks), vec);
  return hipGetLastError();
}

}  // namespace llmopt
