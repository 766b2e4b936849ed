// The products of many tokens: y = x w^T + bias, and silu(x gate^T) * (x up^T) quantized, in tiles.
//
//   y[m][n] = sum over blocks b of 128 columns: 2^(ex[m][b] + ew[n / 128][b]) sum of cx[m][k] cw[n][k] over the block
//
// which the matrix core takes as it stands: a step of 128 columns has one scale for each of its rows, so no sum is rescaled and the
// codes go from memory to the products through LDS only, never through a register that is not an operand. Bound by the matrix cores
// from some 500 tokens on, at the clock that their power leaves (2.55 PFLOP/s, gated 2.4, against 3.7 from registers for microseconds, and
// 2.67 and 2.94 of the library's product with one scale for all), below that by the weight's way from memory.
//
// A workgroup holds a tile's sums in registers, a wave 128 weight rows x 16 TM tokens of them, and STAGES steps of both operands in
// LDS, loaded past the registers as whole lines of 128 bytes and swizzled (no bank conflicts in any case). What was measured (MI355X, in
// a graph, us; down is 4096 x 14336, gate and up 14336 x 4096 each, of 8192 tokens):
//   products of 16 x 16 straight from memory, a wave each: down 7064, gate and up 15942
//   256 x 256 in eight waves, one barrier a step: 445, 1067
//   loads dealt among the products of two phases, scales of 32 steps at a time in LDS: 383, 765
//   tiles one after the other, the next one's first stages beside the last products and the results' stores: 374, 737
//   maxima within 1e-4 of a border of the scales summed again (f8_common.hpp): 374, 760; within 2^-10, equal tokens once: 377, 782 - 797
//   the bias in LDS with the scales, stores of 16 bytes at any alignment: the same at these sizes; 1536 x 1024 with a bias 38 -> 26, 1536 x 1040 of
//   777 tokens with one 11.3 -> 8.9, 5225 x 2592 of 188 tokens 18.4 -> 13.4
// Level or worse: products of 32 x 32 (387, 799 - 823), waves of 64 rows x 32 or 64 tokens in the smaller tiles (a fifth to a third
// fewer LDS reads, all sizes within 2 %), a prefetch into L2 (443 for 421), waves of higher priority, 1 to 32 token tiles a sweep
// instead of 4 (within 3 %). Without the loads down takes 331, without the LDS reads 357, without either and the barrier 292: that is
// what the clock leaves of the products alone.
#include "f8_common.hpp"
#include "f8_mfma.hpp"

namespace llmopt {
namespace {

constexpr int kStep = kF8Group;  // columns of a step: one scale

// Byte offsets that a buffer load finds behind its buffer's end: zeros.
constexpr uint32_t kOutside = 0x7FFFFFF0u;

constexpr int kChunk = 32;        // steps whose scales are in LDS at a time
constexpr int kScaleRow = kChunk + 4;  // bytes of a row of them (16 rows in 16 banks)

// Stores of 16 bytes take any address that fits their elements.
typedef uint32_t Wide2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t Wide1 __attribute__((ext_vector_type(4), aligned(1)));

// Of an operand's scales, what one thread brings to LDS: a row's bytes of the steps first .. first + 31.
struct ScaleRow {
  uint32_t v[kChunk / 4];
  __device__ __forceinline__ void load(const uint8_t* row, int first, int steps) {
    const int count = steps - first < kChunk ? steps - first : kChunk;
#pragma unroll
    for (int i = 0; i < kChunk / 4; ++i) {
      v[i] = 0;
      if (4 * i + 4 <= count) {
        __builtin_memcpy(&v[i], row + first + 4 * i, 4);
      } else {
#pragma unroll
        for (int e = 0; e < 3; ++e)
          if (4 * i + e < count) v[i] |= uint32_t(row[first + 4 * i + e]) << (8 * e);
      }
    }
  }
  __device__ __forceinline__ void store(uint8_t* to) const {
#pragma unroll
    for (int i = 0; i < kChunk / 4; ++i) reinterpret_cast<uint32_t*>(to)[i] = v[i];
  }
};

template <int WN, int WM, int TM, int STAGES, bool GATED, bool PARTS, class Out>
__global__ void __launch_bounds__(64 * WN * WM) __attribute__((amdgpu_waves_per_eu(2, 2)))
    tiles_kernel(const F8TilesArgs a) {
  constexpr int kWaves = WN * WM;
  constexpr int kRowsN = 128 * WN, kRowsM = 16 * TM * WM;
  constexpr int kWide = GATED ? kRowsN / 2 : kRowsN;  // features of a tile
  constexpr int kStage = (kRowsN + kRowsM) * kStep;
  constexpr int kLoadsN = kRowsN / 8 / kWaves, kLoadsM = kRowsM / 8 / kWaves, kLoads = kLoadsN + kLoadsM;
  static_assert(kLoadsN * 8 * kWaves == kRowsN && kLoadsM * 8 * kWaves == kRowsM, "whole loads for every wave");
  static_assert(64 * kWaves >= kRowsM + 2, "a thread for every row of scales");
  // What a wave stores of a whole tile, at least.
  constexpr int kStores = PARTS ? 8 * TM : GATED ? TM : 4 * TM;
  extern __shared__ __align__(1024) uint8_t lds[];
  uint8_t* const scales = lds + STAGES * kStage;
  uint32_t* const tops = reinterpret_cast<uint32_t*>(scales + (kRowsM + 2) * kScaleRow);  // [2][kRowsM] (gated)
  float* const biases = reinterpret_cast<float*>(tops);  // [kRowsN] (a whole product)
  constexpr bool kBias = !GATED && !PARTS;

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wn = wave % WN, wm = wave / WN;
  const int r = lane & 15, g = lane >> 4;
  auto fence = [] { __builtin_amdgcn_sched_barrier(0); };

  // ---- tiles: workgroup i takes i, i + grid, ... ----
  // Neighbouring workgroups go to different XCDs, so each XCD takes a run of tiles of its own; within it `kSweep` token
  // tiles per sweep over the features, whose operands then meet in its L2.
  const uint32_t tiles = a.tiles_n * a.tiles_m, count = tiles * (PARTS ? a.splits : 1);
  struct Tile {
    uint32_t tn, tm, split;
    int begin, steps;  // its steps of 128 columns
  };
  auto tile_of = [&](uint32_t id) {
    constexpr uint32_t kSweep = 4;
    const uint32_t per = count / 8, rest = count % 8, xcd = id % 8;
    id = xcd * per + min(xcd, rest) + id / 8;
    Tile t;
    t.split = PARTS ? __builtin_amdgcn_readfirstlane(id / tiles) : 0;
    if (PARTS) id -= t.split * tiles;
    const uint32_t in_sweep = kSweep * a.tiles_n, first_m = id / in_sweep * kSweep;
    const uint32_t rows_m = min(a.tiles_m - first_m, kSweep), left = id % in_sweep;
    // (quotients are computed in vector registers; buffers and scalar offsets want scalar ones)
    t.tn = __builtin_amdgcn_readfirstlane(left / rows_m);
    t.tm = __builtin_amdgcn_readfirstlane(first_m + left - left / rows_m * rows_m);
    t.begin = PARTS ? int(t.split * a.steps_per_split) : 0;
    t.steps = PARTS ? min(int(a.steps_per_split), a.steps - t.begin) : a.steps;
    return t;
  };
  auto rows_n_of = [&](const Tile& t) {
    const int64_t left = a.N - int64_t(t.tn) * kWide;
    return left < kWide ? int(left) : kWide;
  };
  auto rows_m_of = [&](const Tile& t) {
    const int64_t left = a.M - int64_t(t.tm) * kRowsM;
    return left < kRowsM ? int(left) : kRowsM;
  };

  // ---- loads: lane l of load j brings 16 bytes of row 8 (..) + l / 8, its chunk l % 8 swizzled ----
  const uint32_t K = uint32_t(a.K);
  struct Source {  // of a tile's stages
    __amdgpu_buffer_rsrc_t w[2], x;
    uint32_t k_end;
  };
  auto source_of = [&](const Tile& t) {
    const int64_t n0 = int64_t(t.tn) * kWide, m0 = int64_t(t.tm) * kRowsM;
    const uint32_t rows_n = uint32_t(rows_n_of(t)), rows_m = uint32_t(rows_m_of(t));
    Source s;
    s.w[0] = make_rsrc(a.w[0].codes + n0 * a.w[0].ld, (rows_n - 1) * uint32_t(a.w[0].ld) + K);
    s.w[1] = make_rsrc(a.w[GATED].codes + n0 * a.w[GATED].ld, (rows_n - 1) * uint32_t(a.w[GATED].ld) + K);
    s.x = make_rsrc(a.x + m0 * a.ldx, (rows_m - 1) * uint32_t(a.ldx) + K);
    s.k_end = PARTS ? min(K, uint32_t(t.begin + t.steps) * kStep) : K;
    return s;
  };
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
  // Loads first .. last - 1 of a stage.
  auto load_stage = [&](const Source& src, int step, uint8_t* buf, int first, int last) {
    const uint32_t k = uint32_t(step) * kStep;
    const bool whole = k + kStep <= src.k_end;  // else columns behind the end are zeros
    // The strides are opaque here, so that offsets are computed where they are used and hold no registers.
    uint32_t ld[3] = {uint32_t(a.w[0].ld), uint32_t(a.w[GATED].ld), uint32_t(a.ldx)};
    asm volatile("" : "+s"(ld[0]), "+s"(ld[1]), "+s"(ld[2]));
#pragma unroll
    for (int j = first; j < last; ++j) {
      if (j < kLoadsN) {
        const bool second = GATED && j >= kHalf;
        uint32_t o = off_n[second] + uint32_t(8 * (second ? j - kHalf : j)) * ld[second] + col_n(j);
        if (!whole) o = k + col_n(j) < src.k_end ? o : kOutside;
        load_lds16_cached(src.w[second], buf + base_n(j) * kStep, o, k);
      } else {
        uint32_t o = off_m + uint32_t(8 * (j - kLoadsN)) * ld[2];
        if (!whole) o = k + col_m < src.k_end ? o : kOutside;
        load_lds16_cached(src.x, buf + (kRowsN + base_m(j - kLoadsN)) * kStep, o, k);
      }
    }
  };
  // A load that finds the queue full holds up its wave, products behind it included; so they are dealt to two phases, between
  // the products.
  constexpr int kSlots = 2 * TM;
  auto load_slot = [&](const Source& src, int step, uint8_t* to, int slot) {
    load_stage(src, step, to, kLoads * slot / kSlots, kLoads * (slot + 1) / kSlots);
  };

  // ---- scales: a chunk of steps at a time in LDS, a row of tokens or of the weight's blocks a thread; the bias with the first ----
  ScaleRow row;  // of the chunk after the one in LDS
  float bias_of = 0.0f;
  auto load_scales = [&](const Tile& t, int first) {
    const int i = threadIdx.x;
    const uint8_t* at = nullptr;
    if (i < kRowsM) {
      at = a.x_scales + (int64_t(t.tm) * kRowsM + min(i, rows_m_of(t) - 1)) * a.ldxs;
    } else if (i < kRowsM + (GATED ? 2 : WN)) {
      const int second = i - kRowsM;
      if (GATED)
        at = a.w[second].scales + t.tn * a.w[second].lds;
      else
        at = a.w[0].scales + min(t.tn * WN + second, uint32_t((a.N - 1) / kF8Group)) * a.w[0].lds;
    }
    if (at) row.load(at, t.begin + first, t.begin + t.steps);
    if constexpr (kBias) {
      const int64_t n = int64_t(t.tn) * kWide + i;
      if (a.bias && first == 0 && i < kRowsN) bias_of = n < a.N ? Out::load(static_cast<const typename Out::raw*>(a.bias)[n]) : 0.0f;
    }
  };
  auto store_scales = [&] {
    wait_lgkmcnt0();
    __builtin_amdgcn_s_barrier();  // the chunk before this one has been read
    if (threadIdx.x < kRowsM + 2) row.store(scales + threadIdx.x * kScaleRow);
    if (kBias && threadIdx.x < kRowsN) biases[threadIdx.x] = bias_of;
    wait_lgkmcnt0();
    __builtin_amdgcn_s_barrier();
    fence();
  };
  const uint8_t* const sx_at = scales + (wm * TM * 16 + r) * kScaleRow;
  const uint8_t* const sw_at = scales + (kRowsM + (GATED ? 0 : wn)) * kScaleRow;
  uint32_t sx[TM], sw[2], sx_next[TM], sw_next[2];
  auto read_scales = [&](int step, uint32_t* x, uint32_t* w) {
    step %= kChunk;
#pragma unroll
    for (int u = 0; u < TM; ++u) x[u] = sx_at[u * 16 * kScaleRow + step];
    w[0] = sw_at[step];
    if (GATED) w[1] = sw_at[kScaleRow + step];
  };

  // ---- fragments ----
  // The weight's rows are dealt to the matrix core so that a lane's sums of its 8 tiles are neighbours: lane (r, g) gets rows
  // 32 g + 4 t + i of the wave's 128 in tile t, element i (gated: 16 g + 4 t + i of the gate's 64, then of up's).
  const int row_n = GATED ? wn * 64 + (r >> 2) * 16 + (r & 3) : wn * 128 + (r >> 2) * 32 + (r & 3);
  uint32_t at_n = row_n * kStep + 16 * (g ^ (r & 7)), at_m = (kRowsN + wm * TM * 16 + r) * kStep + 16 * (g ^ (r & 7));
  auto frag = [&](uint32_t at, int offset) {
    const u32x4 lo = *reinterpret_cast<const u32x4*>(lds + at + offset);
    const u32x4 hi = *reinterpret_cast<const u32x4*>(lds + (at ^ 64) + offset);
    return __builtin_bit_cast(i32x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  };
  auto frag_n = [&](int t) { return frag(at_n, (GATED ? (t >> 2) * kWide + (t & 3) * 4 : t * 4) * kStep); };
  auto frag_m = [&](int u) { return frag(at_m, u * 16 * kStep); };

  // ---- products ----
  // A step's 8 TM products are dealt to four phases of two weight tiles. In each, the weight tiles of the next phase come from
  // LDS. In front of the last phase everything of this step is in registers and the next stage in LDS (a barrier), so that
  // phase brings in the next step's first fragments, each token tile's when its registers have served, and starts the loads
  // of STAGES stages on into this step's buffer. A turn of the loop is a step's last phase and the next one's first three; it
  // has no branch: the compiler would move products behind it.
  f32x4 acc[8][TM];
  i32x8 b[TM], w[4];
  uint32_t buf = 0;  // of the step
  auto mul = [&](int t, int u) { acc[t][u] = mfma_f8(w[t & 3], b[u], acc[t][u], sw[GATED ? t >> 2 : 0], sx[u]); };
  auto advance = [&] {
    const uint32_t next = buf == (STAGES - 1) * kStage ? 0u : buf + kStage;
    at_n += next - buf, at_m += next - buf, buf = next;
  };
  auto phases = [&](auto&& between) {  // the first three of a step
#pragma unroll
    for (int phase = 0; phase < 3; ++phase) {
      const int t = 2 * phase;
#pragma unroll
      for (int u = 0; u < TM; ++u) {
        if (u == 0) w[(t + 2) & 3] = frag_n(t + 2);
        if (u == TM / 2) w[(t + 3) & 3] = frag_n(t + 3);
        mul(t, u);
        if (phase == 0) between(u);
        mul(t + 1, u);
        fence();
      }
    }
  };
  // Step s's last phase and step s + 1's others; at most OPEN of the loads and stores issued so far may be under way in front of
  // it. The stage `load` of `src` is loaded (zeros behind its end).
  auto turn = [&](int s, const Source& src, int load, auto open) {
    read_scales(s + 1, sx_next, sw_next);
    wait_lgkmcnt0();
    wait_vmcnt<decltype(open)::value>();
    __builtin_amdgcn_s_barrier();
    fence();
    uint8_t* const freed = lds + buf;
    advance();
    fence();
#pragma unroll
    for (int u = 0; u < TM; ++u) {
      if (u == 0) w[0] = frag_n(0);
      if (u == TM / 2) w[1] = frag_n(1);
      mul(6, u);
      load_slot(src, load, freed, u);
      mul(7, u);
      fence();
      b[u] = frag_m(u);
    }
#pragma unroll
    for (int u = 0; u < TM; ++u) sx[u] = sx_next[u];
    sw[0] = sw_next[0];
    if (GATED) sw[1] = sw_next[1];
    fence();
    phases([&](int u) { load_slot(src, load, freed, TM + u); });
  };

  uint32_t id = blockIdx.x;
  Tile tile = tile_of(id);
  Source source = source_of(tile);  // of the stages that are loaded
#pragma unroll
  for (int i = 0; i < STAGES; ++i) load_stage(source, tile.begin + i, lds + i * kStage, 0, kLoads);
  load_scales(tile, 0);
  wait_vmcnt<0>();
  bool stored = false;  // a whole tile's results after the loads of this one's stages
  for (;;) {
    // The tile after this one, whose first stages follow this one's last (there are more than STAGES steps then).
    const bool more = id + gridDim.x < count;
    const Tile next = more ? tile_of(id + gridDim.x) : tile;

    store_scales();  // (and a barrier)
    if (tile.steps > kChunk)
      load_scales(tile, kChunk);
    else if (more)
      load_scales(next, 0);
    read_scales(0, sx, sw);
#pragma unroll
    for (int u = 0; u < TM; ++u) b[u] = frag_m(u);
    w[0] = frag_n(0);
    w[1] = frag_n(1);
#pragma unroll
    for (int t = 0; t < 8; ++t)
#pragma unroll
      for (int u = 0; u < TM; ++u) acc[t][u] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    fence();
    phases([](int) {});

    const int last = tile.steps - 1, own = max(0, tile.steps - STAGES);  // from turn `own` on the next tile's stages are loaded
    int load = tile.begin + STAGES;
    // The stages that a turn waits for were loaded in front of the results' stores.
    if (own > 0 && stored) turn(0, source, load++, std::integral_constant<int, (STAGES - 2) * kLoads + kStores>{});
    for (int s = load - tile.begin - STAGES; s < last;) {
      if ((s + 1) % kChunk == 0) {
        store_scales();
        if (s + 1 + kChunk < tile.steps)
          load_scales(tile, s + 1 + kChunk);
        else if (more)
          load_scales(next, 0);
      }
      if (s == own) {
        source = source_of(next), load = next.begin;
        if (!more) source.k_end = 0;
      }
      const int end = min(s < own ? own : last, (s + 1) / kChunk * kChunk + kChunk - 1);
#pragma unroll 1
      for (; s < end; ++s) turn(s, source, load++, std::integral_constant<int, (STAGES - 2) * kLoads>{});
    }
    wait_lgkmcnt0();
    __builtin_amdgcn_s_barrier();  // the last stage is in registers
    fence();
#pragma unroll
    for (int u = 0; u < TM; ++u) {
      mul(6, u);
      mul(7, u);
    }
    // All that was loaded so far has to be here before the next tile begins: the scales and its stages but the last. It is
    // waited for now, while no stores are under way.
    wait_vmcnt<0>();
#pragma unroll
    for (uint32_t& v : row.v) asm volatile("" : "+v"(v));
    if constexpr (kBias) asm volatile("" : "+v"(bias_of));
    fence();
    if (last <= own) {  // a walk of one step, or none that the next tile's stages begin in
      source = source_of(next), load = next.begin;
      if (!more) source.k_end = 0;
    }
    load_stage(source, load, lds + buf, 0, kLoads);
    advance();
    fence();

    // ---- results ----
    const int64_t n0 = int64_t(tile.tn) * kWide, m0 = int64_t(tile.tm) * kRowsM;
    const int rows_n = rows_n_of(tile);
    if constexpr (PARTS) {  // rows of a multiple of 16 features
      const int64_t n = n0 + wn * 128 + 32 * g;
#pragma unroll
      for (int u = 0; u < TM; ++u) {
        const int64_t m = m0 + (wm * TM + u) * 16 + r;
        if (m >= a.M) continue;
        float* out = a.parts + (int64_t(tile.split) * a.M + m) * a.ld_parts + n;
#pragma unroll
        for (int t = 0; t < 8; ++t)
          if (n + 4 * t < a.N) *reinterpret_cast<f32x4*>(out + 4 * t) = acc[t][u];
      }
    } else if constexpr (!GATED) {
      using Raw = typename Out::raw;
      const int64_t n = n0 + wn * 128 + 32 * g;
      const bool bias = a.bias != nullptr;
#pragma unroll
      for (int u = 0; u < TM; ++u) {
        const int64_t m = m0 + (wm * TM + u) * 16 + r;
        if (m >= a.M) continue;
        Raw* y = static_cast<Raw*>(a.y) + m * a.ldy;
#pragma unroll
        for (int t = 0; t < 8; t += 2) {
          float v[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = acc[t + i / 4][u][i & 3];
          if (bias) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] += biases[wn * 128 + 32 * g + 4 * t + i];
          }
          u32x4 out;
#pragma unroll
          for (int i = 0; i < 4; ++i) out[i] = pack16<Out>(v[2 * i], v[2 * i + 1]);
          if (n + 4 * t + 8 <= a.N) {
            *reinterpret_cast<Wide2*>(y + n + 4 * t) = out;
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
              if (n + 4 * t + i < a.N) y[n + 4 * t + i] = Raw(out[i >> 1] >> (16 * (i & 1)));
          }
        }
      }
    } else {
      // A group's 128 features lie in two waves, 16 in a lane: the largest magnitude goes across lanes and through LDS.
      float v[TM][16];
      uint32_t top[TM];
      const int f0 = wn * 64 + 16 * g;
      const int64_t m = m0 + wm * TM * 16 + r;
#pragma unroll
      for (int u = 0; u < TM; ++u) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float gate = acc[i >> 2][u][i & 3], up = acc[4 + (i >> 2)][u][i & 3];
          v[u][i] = f0 + i < rows_n ? f8_swiglu(gate, up) : 0.0f;
        }
        uint32_t most = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) most = max(most, magnitude(v[u][i]));
        most = max(most, uint32_t(__shfl_xor(int(most), 16, 64)));
        most = max(most, uint32_t(__shfl_xor(int(most), 32, 64)));
        top[u] = m + 16 * u < a.M ? most : 0u;
      }
      // (The arguments are read anew, where they are needed at all: no registers hold them beside the products.)
      auto* args = (const F8TilesArgs*)__builtin_amdgcn_kernarg_segment_ptr();
      asm volatile("" : "+s"(args));
      f8_settle<false, 15>([&] { return F8Gated{args->x, args->ldx, args->x_scales, args->ldxs, {args->w[0], args->w[1]}, args->K}; }, v, top, m, n0 + f0);
#pragma unroll
      for (int u = 0; u < TM; ++u)
        if (g == 0) tops[wn * kRowsM + (wm * TM + u) * 16 + r] = top[u];
      wait_lgkmcnt0();
      __builtin_amdgcn_s_barrier();
#pragma unroll
      for (int u = 0; u < TM; ++u) {
        const int at = (wm * TM + u) * 16 + r;
        const int64_t m = m0 + at;
        if (m >= a.M) continue;
        const uint32_t scale = f8_scale(max(tops[at], tops[kRowsM + at]));
        const float inv = f8_inverse(scale);
        if (wn == 0 && g == 0) a.scales[m * a.lds + tile.tn] = uint8_t(scale);
        u32x4 out;
#pragma unroll
        for (int i = 0; i < 4; ++i) out[i] = f8_codes4(v[u][4 * i], v[u][4 * i + 1], v[u][4 * i + 2], v[u][4 * i + 3], inv);
        uint8_t* to = a.codes + m * a.ldc + n0 + f0;
        if (f0 + 16 <= rows_n) {
          *reinterpret_cast<Wide1*>(to) = out;
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (f0 + i < rows_n) to[i] = uint8_t(out[i >> 2] >> (8 * (i & 3)));
        }
      }
    }
    if (!more) break;
    stored = rows_n == kWide && m0 + kRowsM <= a.M;
    tile = next, id += gridDim.x;
  }
  wait_vmcnt<0>();  // zeros on their way into LDS
}

template <int WN, int WM, int TM, int STAGES, bool GATED, bool PARTS, class Out>
hipError_t launch(const F8TilesArgs& a, hipStream_t stream) {
  constexpr int kRowsN = 128 * WN, kRowsM = 16 * TM * WM;
  constexpr int kBytes = STAGES * (kRowsN + kRowsM) * kStep + (kRowsM + 2) * kScaleRow + (GATED ? 8 * kRowsM : PARTS ? 0 : 4 * kRowsN);
  static_assert(kBytes <= 160 * 1024, "stages and scales fit LDS");
  auto* kernel = tiles_kernel<WN, WM, TM, STAGES, GATED, PARTS, Out>;
  if constexpr (kBytes > 64 * 1024) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, kBytes);
    if (e != hipSuccess) return e;
  }
  // As many workgroups as the chip holds, each with its tiles one after the other: the next one's first stages are loaded, and
  // this one's results stored, beside the products. Walks too short for that: a workgroup for each tile.
  const uint32_t count = a.tiles_n * a.tiles_m * (PARTS ? a.splits : 1), held = 256 * (kBytes <= 80 * 1024 ? 2 : 1);
  const int shortest = PARTS ? a.steps - int((a.splits - 1) * a.steps_per_split) : a.steps;
  const uint32_t grid = shortest > STAGES && count > held ? held : count;
  hipLaunchKernelGGL(kernel, dim3(grid), dim3(64 * WN * WM), kBytes, stream, a);
  return hipGetLastError();
}

template <int WN, int WM, int TM, int STAGES>
hipError_t launch_shape(F8TilesArgs a, int out_dtype, hipStream_t stream) {
  constexpr int kRowsN = 128 * WN, kRowsM = 16 * TM * WM;
  const bool gated = a.w[1].codes != nullptr;
  const int64_t wide = gated ? kRowsN / 2 : kRowsN;
  a.tiles_n = uint32_t((a.N + wide - 1) / wide);
  a.tiles_m = uint32_t((a.M + kRowsM - 1) / kRowsM);
  a.steps = int((a.K + kStep - 1) / kStep);
  // What no kernel here is for: a grid of such would be of tiles or steps that are not there.
  if (gated ? WN != 2 || a.splits > 1 : a.splits > 1 && (kRowsM == 256 || (a.splits - 1) * a.steps_per_split >= uint32_t(a.steps)))
    return hipErrorInvalidValue;
  if constexpr (kRowsM < 256) {
    if (a.splits > 1) {
      const hipError_t err = launch<WN, WM, TM, STAGES, false, true, ActBf16>(a, stream);
      if (err != hipSuccess) return err;
      return launch_f8_join({a.parts, a.splits, a.M, a.N, a.ld_parts, a.bias, a.y, a.ldy}, out_dtype, stream);
    }
  }
  if constexpr (WN == 2) {
    if (gated) return launch<WN, WM, TM, STAGES, true, false, ActBf16>(a, stream);
  }
  if (out_dtype == kDtF16) return launch<WN, WM, TM, STAGES, false, false, ActF16>(a, stream);
  return launch<WN, WM, TM, STAGES, false, false, ActBf16>(a, stream);
}

}  // namespace

hipError_t launch_f8_tiles(const F8TilesArgs& a, F8Shape shape, int out_dtype, hipStream_t stream) {
  switch (shape) {
    case F8Shape::k256x256: return launch_shape<2, 4, 4, 2>(a, out_dtype, stream);
    case F8Shape::k256x128: return launch_shape<2, 4, 2, 3>(a, out_dtype, stream);
    case F8Shape::k256x64: return launch_shape<2, 4, 1, 3>(a, out_dtype, stream);
    case F8Shape::k128x128: return launch_shape<1, 4, 2, 2>(a, out_dtype, stream);
    default: return launch_shape<1, 4, 1, 3>(a, out_dtype, stream);
  }
}

}  // namespace llmopt
