// The products of many tokens: y = x w^T + bias, and silu(x gate^T) * (x up^T) quantized, in tiles.
#include "f8_common.hpp"
#include "f8_mfma.hpp"

namespace llmopt {
namespace {

constexpr int kStep = kF8Group;  // columns of a step: one scale

// Byte offsets that a buffer load finds behind its buffer's end: zeros.
constexpr uint32_t kOutside = 0x7FFFFFF0u;

template <int WN, int WM, int TM, bool GATED, class Out>
__global__ void __launch_bounds__(64 * WN * WM) __attribute__((amdgpu_waves_per_eu(2, 2)))
    tiles_kernel(const F8TilesArgs a) {
  constexpr int kWaves = WN * WM;
  constexpr int kRowsN = 128 * WN, kRowsM = 16 * TM * WM;
  constexpr int kStage = (kRowsN + kRowsM) * kStep;
  constexpr uint32_t kBuffer = kStage <= 32768 ? 32768 : 65536;  // from one stage's buffer to the other's
  static_assert(kStage <= 65536, "two stages in LDS");
  constexpr int kLoadsN = kRowsN / 8 / kWaves, kLoadsM = kRowsM / 8 / kWaves;
  static_assert(kLoadsN * 8 * kWaves == kRowsN && kLoadsM * 8 * kWaves == kRowsM, "whole loads for every wave");
  extern __shared__ __align__(1024) uint8_t lds[];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wn = wave % WN, wm = wave / WN;
  const int r = lane & 15, g = lane >> 4;

  // Tile order: neighbouring workgroups go to different XCDs, so each XCD takes a run of tiles of its own; within it
  // `kSweep` token tiles per sweep over the features, whose operands then meet in its L2.
  constexpr uint32_t kSweep = 4;
  uint32_t id = blockIdx.x;
  const uint32_t count = gridDim.x;
  {
    const uint32_t per = count / 8, rest = count % 8, xcd = id % 8, at = id / 8;
    id = xcd * per + min(xcd, rest) + at;
  }
  const uint32_t in_sweep = kSweep * a.tiles_n;
  const uint32_t first_m = id / in_sweep * kSweep;
  const uint32_t rows_m = min(a.tiles_m - first_m, kSweep);
  const uint32_t left = id % in_sweep;
  // (quotients are computed in vector registers; buffers and scalar offsets want scalar ones)
  const uint32_t tn = __builtin_amdgcn_readfirstlane(left / rows_m);
  const uint32_t tm = __builtin_amdgcn_readfirstlane(first_m + left - left / rows_m * rows_m);
  const int64_t m0 = int64_t(tm) * kRowsM;
  const int64_t n0 = int64_t(tn) * (GATED ? kRowsN / 2 : kRowsN);

  // ---- loads: lane l of load j brings 16 bytes of row 8 (..) + l / 8, its chunk l % 8 swizzled ----
  constexpr int kWide = GATED ? kRowsN / 2 : kRowsN;  // features of a tile
  const int rows_n = a.N - n0 < kWide ? int(a.N - n0) : kWide, rows_mm = a.M - m0 < kRowsM ? int(a.M - m0) : kRowsM;
  const uint32_t K = uint32_t(a.K);
  const auto wq0 = make_rsrc(a.w[0].codes + n0 * a.w[0].ld, uint32_t(rows_n - 1) * uint32_t(a.w[0].ld) + K);
  const auto wq1 = make_rsrc(a.w[GATED].codes + n0 * a.w[GATED].ld, uint32_t(rows_n - 1) * uint32_t(a.w[GATED].ld) + K);
  const auto xq = make_rsrc(a.x + m0 * a.ldx, uint32_t(rows_mm - 1) * uint32_t(a.ldx) + K);
  // LDS row of load j's first lane; the chunk that a lane brings: its own position swizzled by its row.
  constexpr int kShift = GATED ? 4 : 5, kHalf = kLoadsN / 2;
  auto base_n = [&](int j) {
    return GATED ? (j < kHalf ? 0 : kWide) + 8 * (wave * kHalf + j % kHalf) : 8 * (wave * kLoadsN + j);
  };
  auto base_m = [&](int j) { return 8 * (wave * kLoadsM + j); };
  auto col_n = [&](int j) { return 16u * ((lane & 7) ^ (((lane >> 3) & 3) | ((base_n(j) >> kShift & 1) << 2))); };
  const uint32_t col_m = 16u * ((lane & 7) ^ (lane >> 3));
  // Offsets of the first load's rows; the next one's are eight rows on. Rows behind the operand's last are behind the buffer's
  // end, and read as zeros.
  uint32_t off_n[2];
  off_n[0] = uint32_t(base_n(0) + lane / 8) * uint32_t(a.w[0].ld);
  off_n[1] = uint32_t(base_n(0) + lane / 8) * uint32_t(a.w[GATED].ld);
  const uint32_t off_m = uint32_t(base_m(0) + lane / 8) * uint32_t(a.ldx) + col_m;
  auto load_stage = [&](int step, uint8_t* buf) {
    const uint32_t k = uint32_t(step) * kStep;
    const bool whole = k + kStep <= K;  // else columns behind the end are zeros
    // The strides are opaque here, so that offsets are computed where they are used and hold no registers.
    uint32_t ld[3] = {uint32_t(a.w[0].ld), uint32_t(a.w[GATED].ld), uint32_t(a.ldx)};
    asm volatile("" : "+s"(ld[0]), "+s"(ld[1]), "+s"(ld[2]));
#pragma unroll
    for (int j = 0; j < kLoadsN; ++j) {
      const bool second = GATED && j >= kHalf;
      uint32_t o = off_n[second] + uint32_t(8 * (second ? j - kHalf : j)) * ld[second] + col_n(j);
      if (!whole) o = k + col_n(j) < K ? o : kOutside;
      load_lds16_cached(second ? wq1 : wq0, buf + base_n(j) * kStep, o, k);
    }
#pragma unroll
    for (int j = 0; j < kLoadsM; ++j) {
      uint32_t o = off_m + uint32_t(8 * j) * ld[2];
      if (!whole) o = k + col_m < K ? o : kOutside;
      load_lds16_cached(xq, buf + (kRowsN + base_m(j)) * kStep, o, k);
    }
  };

  // ---- scales ----
  const auto xs = make_rsrc(a.x_scales + m0 * a.ldxs, uint32_t(rows_mm - 1) * uint32_t(a.ldxs) + uint32_t(a.steps));
  const uint32_t xs_off = uint32_t(wm * TM * 16 + r) * uint32_t(a.ldxs);
  const uint32_t ws_row = GATED ? tn : min(tn * WN + wn, uint32_t((a.N - 1) / kF8Group));
  const auto ws0 = make_rsrc(a.w[0].scales + ws_row * a.w[0].lds, uint32_t(a.steps));
  const auto ws1 = make_rsrc(a.w[GATED].scales + ws_row * a.w[GATED].lds, uint32_t(a.steps));
  uint32_t sx[TM], sw[2], sx_next[TM], sw_next[2];
  auto load_scales = [&](int step, uint32_t* x, uint32_t* w) {
    uint32_t ld = uint32_t(a.ldxs);
    asm volatile("" : "+s"(ld));
#pragma unroll
    for (int t = 0; t < TM; ++t) x[t] = __builtin_amdgcn_raw_buffer_load_b8(xs, int(xs_off + uint32_t(16 * t) * ld), step, 0);
    w[0] = __builtin_amdgcn_raw_buffer_load_b8(ws0, 0, step, 0);
    if (GATED) w[1] = __builtin_amdgcn_raw_buffer_load_b8(ws1, 0, step, 0);
  };

  // ---- fragments ----
  // The weight's rows are dealt to the matrix core so that a lane's sums of its 8 tiles are neighbours: lane (r, g) gets rows
  // 32 g + 4 t + i of the wave's 128 in tile t, element i (gated: 16 g + 4 t + i of the gate's 64, then of up's).
  const int row_n = GATED ? wn * 64 + (r >> 2) * 16 + (r & 3) : wn * 128 + (r >> 2) * 32 + (r & 3);
  const int at_n = row_n * kStep + 16 * (g ^ (r & 7)), at_m = (kRowsN + wm * TM * 16 + r) * kStep + 16 * (g ^ (r & 7));
  // Four addresses, of either half of the columns, that turn to the other buffer at each step (a power of two apart).
  uint32_t frag_at[4] = {uint32_t(at_n), uint32_t(at_n ^ 64), uint32_t(at_m), uint32_t(at_m ^ 64)};
  auto frag = [&](int which, int offset) {
    const u32x4 lo = *reinterpret_cast<const u32x4*>(lds + frag_at[which] + offset);
    const u32x4 hi = *reinterpret_cast<const u32x4*>(lds + frag_at[which + 1] + offset);
    return __builtin_bit_cast(i32x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  };
  auto frag_n = [&](int t) { return frag(0, (GATED ? (t >> 2) * kWide + (t & 3) * 4 : t * 4) * kStep); };
  auto frag_m = [&](int u) { return frag(2, u * 16 * kStep); };

  f32x4 acc[8][TM];
#pragma unroll
  for (int t = 0; t < 8; ++t)
#pragma unroll
    for (int u = 0; u < TM; ++u) acc[t][u] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  // A step's 32 (8 TM) products are dealt to four phases of two weight tiles. In each, the weight tiles of the next phase come
  // from LDS. In front of the last phase everything of this step is in registers and the next stage in LDS (a barrier), so
  // that phase brings in the next step's first fragments, each token tile's when its registers have served, and starts the
  // loads of the stage after the next into this step's buffer.
  i32x8 b[TM], w[4];
  auto fence = [] { __builtin_amdgcn_sched_barrier(0); };
  load_stage(0, lds);
  load_scales(0, sx, sw);
  load_stage(1, lds + kBuffer);
  wait_vmcnt<0>();
  __builtin_amdgcn_s_barrier();
  fence();
#pragma unroll
  for (int u = 0; u < TM; ++u) b[u] = frag_m(u);
  w[0] = frag_n(0);
  w[1] = frag_n(1);
  auto mul = [&](int t, int u) { acc[t][u] = mfma_f8(w[t & 3], b[u], acc[t][u], sw[GATED ? t >> 2 : 0], sx[u]); };
#pragma unroll 1
  for (int s = 0; s < a.steps; ++s) {
    load_scales(s + 1, sx_next, sw_next);  // (zeros behind the end)
    fence();
#pragma unroll
    for (int phase = 0; phase < 3; ++phase) {
      const int t = 2 * phase;
#pragma unroll
      for (int u = 0; u < TM; ++u) {
        if (u == 0) w[(t + 2) & 3] = frag_n(t + 2);
        if (u == TM / 2) w[(t + 3) & 3] = frag_n(t + 3);
        mul(t, u);
        mul(t + 1, u);
        fence();
      }
    }
    wait_lgkmcnt0();
    wait_vmcnt<0>();
    __builtin_amdgcn_s_barrier();
    fence();
#pragma unroll
    for (int i = 0; i < 4; ++i) frag_at[i] ^= kBuffer;
    load_stage(s + 2, lds + (s & 1) * kBuffer);  // (zeros behind the end)
    fence();
#pragma unroll
    for (int u = 0; u < TM; ++u) {
      if (u == 0) w[0] = frag_n(0);
      if (u == TM / 2) w[1] = frag_n(1);
      mul(6, u);
      mul(7, u);
      fence();
      b[u] = frag_m(u);
    }
#pragma unroll
    for (int u = 0; u < TM; ++u) sx[u] = sx_next[u];
    sw[0] = sw_next[0];
    if (GATED) sw[1] = sw_next[1];
    fence();
  }

  // ---- results ----
  if constexpr (!GATED) {
    using Raw = typename Out::raw;
    const int64_t n = n0 + wn * 128 + 32 * g;
    const Raw* bias = static_cast<const Raw*>(a.bias);
#pragma unroll
    for (int u = 0; u < TM; ++u) {
      const int64_t m = m0 + (wm * TM + u) * 16 + r;
      if (m >= a.M) continue;
      Raw* y = static_cast<Raw*>(a.y) + m * a.ldy;
#pragma unroll
      for (int t = 0; t < 8; t += 2) {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          v[i] = acc[t + i / 4][u][i & 3];
          const int64_t at = n + 4 * t + i;
          if (bias && at < a.N) v[i] += Out::load(bias[at]);
        }
        u32x4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = uint32_t(Out::store(v[2 * i])) | (uint32_t(Out::store(v[2 * i + 1])) << 16);
        if (a.vec && n + 4 * t + 8 <= a.N) {
          *reinterpret_cast<u32x4*>(y + n + 4 * t) = w;
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (n + 4 * t + i < a.N) y[n + 4 * t + i] = Raw(w[i >> 1] >> (16 * (i & 1)));
        }
      }
    }
  } else {
    // A group's 128 features lie in two waves, 16 in a lane: the largest magnitude goes across lanes and through LDS.
    wait_lgkmcnt0();
    __syncthreads();
    uint32_t* tops = reinterpret_cast<uint32_t*>(lds);  // [2][kRowsM]
    float v[TM][16];
    uint32_t top[TM];
    const int f0 = wn * 64 + 16 * g;
#pragma unroll
    for (int u = 0; u < TM; ++u) {
      top[u] = 0;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float gate = acc[i >> 2][u][i & 3], up = acc[4 + (i >> 2)][u][i & 3];
        v[u][i] = f0 + i < rows_n ? gate / (1.0f + __expf(-gate)) * up : 0.0f;
        top[u] = max(top[u], magnitude(v[u][i]));
      }
      top[u] = max(top[u], uint32_t(__shfl_xor(int(top[u]), 16, 64)));
      top[u] = max(top[u], uint32_t(__shfl_xor(int(top[u]), 32, 64)));
      if (g == 0) tops[wn * kRowsM + (wm * TM + u) * 16 + r] = top[u];
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < TM; ++u) {
      const int row = (wm * TM + u) * 16 + r;
      const int64_t m = m0 + row;
      if (m >= a.M) continue;
      const uint32_t scale = f8_scale(max(tops[row], tops[kRowsM + row]));
      const float inv = f8_inverse(scale);
      if (wn == 0 && g == 0) a.scales[m * a.lds + n0 / kF8Group] = uint8_t(scale);
      u32x4 w;
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = f8_codes4(v[u][4 * i], v[u][4 * i + 1], v[u][4 * i + 2], v[u][4 * i + 3], inv);
      uint8_t* out = a.codes + m * a.ldc + n0 + f0;
      if (a.vec && f0 + 16 <= rows_n) {
        *reinterpret_cast<u32x4*>(out) = w;
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (f0 + i < rows_n) out[i] = uint8_t(w[i >> 2] >> (8 * (i & 3)));
      }
    }
  }
}

template <int WN, int WM, int TM, bool GATED, class Out>
hipError_t launch(F8TilesArgs a, hipStream_t stream) {
  constexpr int kRowsN = 128 * WN, kRowsM = 16 * TM * WM;
  a.tiles_n = uint32_t((a.N + (GATED ? kRowsN / 2 : kRowsN) - 1) / (GATED ? kRowsN / 2 : kRowsN));
  a.tiles_m = uint32_t((a.M + kRowsM - 1) / kRowsM);
  a.steps = int((a.K + kStep - 1) / kStep);
  constexpr int kStage = (kRowsN + kRowsM) * kStep;
  constexpr int kBytes = (kStage <= 32768 ? 32768 : 65536) + kStage;
  auto* kernel = tiles_kernel<WN, WM, TM, GATED, Out>;
  static const hipError_t ready = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, kBytes);
  if (ready != hipSuccess) return ready;
  hipLaunchKernelGGL(kernel, dim3(a.tiles_n * a.tiles_m), dim3(64 * WN * WM), kBytes, stream, a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_f8_tiles(const F8TilesArgs& a, int out_dtype, hipStream_t stream) {
  if (a.M == 0 || a.N == 0) return hipSuccess;
  if (a.w[1].codes) return launch<2, 4, 4, true, ActBf16>(a, stream);
  if (out_dtype == kDtF16) return launch<2, 4, 4, false, ActF16>(a, stream);
  return launch<2, 4, 4, false, ActBf16>(a, stream);
}

}  // namespace llmopt
