// Causal attention of many query rows, for packed prompts (16-bit keys and values, rows of a tensor) and for chunks
// over the 8-bit cache (codes by block table). One kernel, two sources of key tiles.
//
// A workgroup of four waves owns 128 query rows of one (sequence, KV head): the sequence's rows are its tokens x the
// `group` query heads that share the KV head, token-major, 32 rows per wave. It walks the keys in tiles of 64, held as
// 16-bit rows in a double buffer in LDS that all rows read:
//   * packed: by direct loads, one tile ahead;
//   * codes: loaded into registers one tile ahead, dequantized to bf16 behind the tile's products (code x power of two:
//     exactly; code x another scale: rounded), and stored.
// Per tile and wave, on v_mfma_f32_32x32x16:
//   * S^T = K Q^T (A: 32 keys x 16 dims from LDS, B: 16 dims x 32 rows, in registers): lane l holds row l % 32
//     against 16 keys of each block of 32 -- keys 8 q + 4 (l / 32) + r --, so a row's softmax takes one exchange
//     between the lane halves;
//   * online softmax in fp32, in powers of two;
//   * O^T += V^T P^T with the probabilities as they lie (slot 4 a + r of lane half h is key 8 a + 4 h + r), V^T by
//     transposing LDS reads of the row-major V tile.
// Bound by the matrix units and the power they draw: the clock falls to 1.65 - 1.94 GHz under it (1.5 - 1.9 under a large
// library product of 1206 TFLOP/s), and MFMAs are under way in half of the cycles, VALU work (32 exponentials, 32 fused
// multiply-adds, 32 roundings and sums per 32 MFMAs) beside them from the SIMD's other wave. Measured (MI355X, heads
// of 128, 32 query and 8 KV heads): one prompt of 8192 in bf16 534 us (1030 TFLOP/s), 4 of 2048 162 (850), 32 of 512 115
// (601). Short prompts: rows, tokens and finiteness by few instructions at a walk's ends (32 of 1 - 1024 tokens in fp16 175 ->
// 165, 512 of 32 106 -> 85), half a tile where the last one has up to 32 keys (165 -> 162). Measured and not taken: 64
// rows per wave (733 against 560 for 8192), eight waves per workgroup (533 against 547, but 199 against 188 for
// 32 prompts), three buffers (575), the next tile's products between the softmax of this one (545 - 576 against 542), three
// workgroups per CU with one V buffer (552 against 545).
// A key that is masked for some rows of a tile only has probability 0 for them, but 0 x infinity would still reach
// their output: a wave whose rows come out with anything that is not finite computes those rows once more, key by
// key (never for finite inputs). That is right but slow: a NaN in the first token of a prompt of 4096 sends all of its rows there,
// 26 ms for 0.17 (of 1024 tokens 5.4, of 512 2.6).
#pragma once

#include <type_traits>

#include "attn_common.hpp"

namespace llmopt {
namespace tile {

enum : int { kSrcPacked = 0, kSrcCodes = 1 };

constexpr int kKeys = 64;
constexpr int kWaves = 4;             // of a workgroup
constexpr int kRows = 32 * kWaves;    // query rows of a workgroup
constexpr float kLog2e = 1.44269504088896340736f;
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));

template <int N>
using Blocks = std::integral_constant<int, N>;

template <bool F16>
struct Op {
  __device__ static f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
    if constexpr (F16)
      return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else
      return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
  __device__ static uint32_t pack(float lo, float hi) {
    if constexpr (F16)
      return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_t{lo, hi}), f16x2_t));  // one instruction
    else
      return pack_bf16(lo, hi);
  }
  __device__ static float add_pair(uint32_t pair, float sum) {  // sum + both halves, in fp32
    if constexpr (F16)
      return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2_t, pair), __builtin_bit_cast(f16x2_t, 0x3C003C00u), sum, false);
    else
      return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, pair), __builtin_bit_cast(bf16x2_t, 0x3F803F80u), sum, false);
  }
};

// Four 16-bit elements of one column of four rows: of 16 lanes, lane 4 r + c reads dims 4 c .. of row r and lane i
// receives dim i of rows 0 .. 3.
__device__ __forceinline__ u32x2 read_transposed(const uint8_t* p) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p));
}

__device__ __forceinline__ float other_half_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float other_half_sum(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Place of 16-byte chunk c within row r of a K or V tile: 16 rows of one K chunk, and the four rows of a transposing
// read of V, fall on distinct banks.
template <int HD>
__device__ __forceinline__ int k_chunk(int r, int c) {
  return HD == 128 ? c ^ (r & 15) : c ^ ((r >> 1) & 7);
}
template <int HD>
__device__ __forceinline__ int v_chunk(int r, int c) {
  return HD == 128 ? c ^ ((r & 3) << 2) : c ^ ((r & 2) << 1);
}

// What a workgroup works on, the same for both sources.
struct Work {
  const void* query;  // its sequence's token 0, its KV head's first query head
  int64_t q_tok_stride, q_head_stride;
  void* out;          // likewise
  int64_t o_tok_stride, o_head_stride;
  int group;
  int rows;   // query rows of the (sequence, KV head)
  int row0;   // the workgroup's first, and its token
  int row0_tok;
  int base;   // position of query token 0
  int t_begin;  // its keys: t_begin (a multiple of 64) <= t < t_end
  int t_end;
  float scale, softcap;
  // packed: key and value rows of the sequence's token 0
  const uint16_t* key;
  const uint16_t* value;
  int64_t k_tok_stride, v_tok_stride;
  int len;
  // codes
  const uint8_t* codes[2];
  const float* scales[2];
  const int32_t* table;
  uint32_t kv_heads, kvh, block_size, ldb, num_blocks;
  // codes: with part_out, the split's normalized rows [rows, HD] and log-sum-exps (powers of two) go there, in fp32
  float* part_out;
  float* part_lse;
};

// KP: 16-bit pieces of a probability. F16: fp16 operands (packed fp16), else bf16. QF16: the
// query's and output's type is fp16 (else bf16). CAP: the scores are soft-capped.
template <int SRC, int FMT, bool F16, bool QF16, int HD, int KP, bool CAP>
__device__ __forceinline__ void attend(const Work& a, uint8_t* lds) {
  constexpr int kCh = HD / 8;               // 16-byte chunks per 16-bit row
  constexpr int kRowBytes = HD * 2;
  constexpr int kTile = kKeys * kRowBytes;  // one K (or V) tile
  constexpr int kRpl = 64 / kCh;            // 16-bit rows per wave load (1 KB)
  constexpr int kTr = kKeys / kWaves;       // rows of a tile that a wave brings in
  constexpr int kLoads = kTr / kRpl;        // packed: in wave loads of K and of V
  constexpr int kCpr = HD / 16;             // codes: 16-byte loads per row
  constexpr int kCrl = 64 / kCpr;           // codes: rows per wave load
  constexpr int kCLoads = kTr / kCrl;
  constexpr int kS = HD / 16;               // 16-dim slices of the scores
  constexpr int kD = HD / 32;               // 32-dim blocks of the output
  // fp16 queries over codes: the keys are the codes themselves, exact in fp16, and their scales, by key in LDS behind
  // the tiles, multiply the scores (two bf16 pieces of the query instead: 287 us against 193 when both were tried, for a chunk of
  // 4 x 512 after up to 3500).
  constexpr bool kRawKeys = SRC == kSrcCodes && QF16;
  static_assert(kLoads > 0 && (SRC == kSrcPacked || kCLoads > 0), "a wave brings in whole loads");
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, half = lane >> 5;
  const uint32_t group = uint32_t(a.group);
  auto tok_of = [&](int row) -> int { return int(uint32_t(row) / group); };
  const int wrow = a.row0 + 32 * wave;  // the wave's first row
  const int own_row = wrow + col;
  const bool row_ok = own_row < a.rows;
  // The token, counted from row0_tok, of the row n rows behind that token's first: (n + 1/2) / group is at least 1 / (2
  // group) away from a whole number, and its three roundings in fp32 are off by less for n < 2^20 (n < group + 128, checked
  // on the host). Integer divisions, here and per row that is loaded or stored, were a third of a short walk's VALU work.
  const float inv_group = __builtin_amdgcn_rcpf(float(a.group));
  const int rem0 = a.row0 - a.row0_tok * a.group + 32 * wave;  // wrow's n
  auto tok_at = [&](int n) -> int { return int((float(n) + 0.5f) * inv_group); };
  const int pos0 = a.base + a.row0_tok;
  const int q_pos = row_ok ? pos0 + tok_at(rem0 + col) : -1;
  const int first_pos = pos0 + __builtin_amdgcn_readfirstlane(tok_at(rem0));
  const int wave_last = wrow < a.rows ? pos0 + __builtin_amdgcn_readfirstlane(tok_at(rem0 + min(31, a.rows - 1 - wrow))) : -1;
  const int first_tile = a.t_begin / kKeys, n_tiles = (a.t_end + kKeys - 1) / kKeys;

  const float neg_inf = -__int_as_float(0x7F800000);
  // Probabilities are 2^(score c - m c), one fma and one exponential per score. c has to be positive for the maximum
  // of the scores to be that of the exponents: a negative scale moves into the query rows, a zero one becomes too
  // small to matter.
  const float magnitude = __builtin_fabsf(a.scale) * kLog2e;
  const float c2 = CAP ? kLog2e : magnitude > 0.0f ? magnitude : 1e-30f;
  const uint32_t q_sign = !CAP && a.scale < 0.0f ? 0x80008000u : 0u;
  const float cap_scale = CAP ? a.scale / a.softcap : 0.0f, cap_exp = cap_scale * (2.0f * kLog2e);
  float m_run = neg_inf, mc = 0.0f, l_run = 0.0f;  // the row's running maximum, m_run c2 (0 without keys), this lane's
                                                   // share of the sum
  f32x16 o[kD];
#pragma unroll
  for (int d = 0; d < kD; ++d)
#pragma unroll
    for (int v = 0; v < 16; ++v) o[d][v] = 0.0f;

  // ---- the wave's query rows: the B operand, dims 16 m + 8 half .. of row col ----
  // The rows come in whole, by direct loads into the second tile buffers (a lane's 16-byte pieces straight from memory
  // would touch each line four times).
  u32x4 qf[kS];
  // Byte offset from row0_tok's first head of row wrow + r; below 2^31 (strides checked on the host).
  auto row_offset = [&](int r, int64_t tok_stride, int64_t head_stride) -> uint32_t {
    const uint32_t n = uint32_t(rem0 + r), t = uint32_t(tok_at(rem0 + r));
    return (n * uint32_t(head_stride) + t * uint32_t(tok_stride - head_stride * a.group)) * 2;
  };
  uint8_t* const q_lds = lds + (wave & 1) * (32 * kRowBytes) + (first_tile & 1 ? 0 : kTile) + (wave >> 1) * (2 * kTile);
  auto fetch_query = [&]() {
    const auto rs = make_rsrc(static_cast<const uint16_t*>(a.query) + a.row0_tok * a.q_tok_stride, 0x7FFFFFFFu);
#pragma unroll
    for (int j = 0; j < 32 / kRpl; ++j) {
      const int r = kRpl * j + lane / kCh;
      // Rows past the end repeat the last one.
      const uint32_t at = row_offset(min(r, a.rows - 1 - wrow), a.q_tok_stride, a.q_head_stride);
      load_lds16_cached(rs, q_lds + kRpl * j * kRowBytes, at + 16 * k_chunk<HD>(r, lane % kCh), 0);
    }
  };
  auto load_query = [&]() {
#pragma unroll
    for (int m = 0; m < kS; ++m) {
      const u32x4 w = *reinterpret_cast<const u32x4*>(q_lds + col * kRowBytes + 16 * k_chunk<HD>(col, 2 * m + half));
      qf[m] = w ^ q_sign;
    }
  };

  // ---- key tiles: two buffers of K and two of V; tile i in buffer i % 2 (offsets: they stay LDS addresses) ----
  auto k_buf = [&](int i) -> uint8_t* { return lds + (i & 1) * kTile; };
  auto v_buf = [&](int i) -> uint8_t* { return lds + 2 * kTile + (i & 1) * kTile; };
  float* const k_scales = reinterpret_cast<float*>(lds + 4 * kTile);  // [2][kKeys], only for kRawKeys
  // Packed: rows past the sequence repeat its last one; no row sees them.
  auto fetch_packed = [&](int k, int i) {
    const int t0 = i * kKeys, last = min(kKeys, a.len - t0) - 1;
    const int64_t stride = k ? a.v_tok_stride : a.k_tok_stride;
    const auto rs = make_rsrc((k ? a.value : a.key) + t0 * stride, uint32_t(last * stride * 2 + kRowBytes));
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      const int r = wave * kTr + kRpl * j + lane / kCh;
      const int c = k ? v_chunk<HD>(r, lane % kCh) : k_chunk<HD>(r, lane % kCh);
      load_lds16_cached(rs, (k ? v_buf(i) : k_buf(i)) + (wave * kTr + kRpl * j) * kRowBytes,
                        uint32_t(min(r, last)) * uint32_t(stride * 2) + 16 * c, 0);
    }
  };
  // Codes: lane l looks up key l of a tile, the table entry some tiles ahead of its use.
  struct Place {
    uint32_t block, row;  // the lane's key: its (block, KV head) and its row of the codes; no key: some row of the cache
    uint64_t mask;        // which keys there are
  };
  struct Held {
    u32x4 codes[kCLoads > 0 ? kCLoads : 1];
    float scale[kCLoads > 0 ? kCLoads : 1];
  };
  struct Look {
    uint32_t bi, slot;  // the key's column in the table, and its slot
  };
  // Tile by tile without dividing again: a tile is tile_blocks blocks and tile_slots slots.
  const uint32_t tile_blocks = SRC == kSrcCodes ? kKeys / a.block_size : 0u;
  const uint32_t tile_slots = kKeys - tile_blocks * a.block_size;
  auto look_at = [&](int i) -> Look {
    const uint32_t t = uint32_t(i * kKeys + lane), bi = t / a.block_size;
    return Look{bi, t - bi * a.block_size};
  };
  auto advance = [&](Look& l) {
    l.slot += tile_slots;
    const bool over = l.slot >= a.block_size;
    l.slot -= over ? a.block_size : 0u;
    l.bi += tile_blocks + (over ? 1u : 0u);
  };
  auto entry_of = [&](int i, const Look& l) -> int32_t {  // t_end is within the table
    return i * kKeys + lane < a.t_end ? a.table[l.bi] : -1;
  };
  auto place_of = [&](const Look& l, int32_t entry) -> Place {
    const bool ok = entry >= 0 && uint32_t(entry) < a.num_blocks;
    const uint32_t block = (ok ? uint32_t(entry) : 0u) * a.kv_heads + a.kvh;
    return Place{block, block * a.block_size + l.slot, __builtin_amdgcn_ballot_w64(ok)};  // below 2^31: checked on the host
  };
  auto fetch_codes = [&](int k, const Place& p) -> Held {
    Held h;
#pragma unroll
    for (int j = 0; j < kCLoads; ++j) {
      const int r = wave * kTr + kCrl * j + lane / kCpr;
      const int64_t block = uint32_t(__shfl(int(p.block), r, 64)), row = uint32_t(__shfl(int(p.row), r, 64));
      h.codes[j] = *reinterpret_cast<const u32x4*>(a.codes[k] + row * HD + 16 * (lane % kCpr));
      h.scale[j] = a.scales[k][block];
    }
    return h;
  };
  auto store_codes = [&](int k, int i, Held& h, uint64_t mask) {
#pragma unroll
    for (int j = 0; j < kCLoads; ++j) {
      const int r = wave * kTr + kCrl * j + lane / kCpr, c = 2 * (lane % kCpr);
      asm("" : "+v"(h.codes[j]));  // whole words until here
      if (k == 1 && mask != ~uint64_t(0) && !((mask >> r) & 1u)) {  // no key: its probability is 0, its value must be finite
        h.codes[j] = u32x4{0u, 0u, 0u, 0u};
        h.scale[j] = 0.0f;
      }
      const float s = h.scale[j];
      if (kRawKeys && k == 0 && lane % kCpr == 0) k_scales[(i & 1) * kKeys + r] = s;
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        u32x4 w;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t x = h.codes[j][2 * q + e];
          if (kRawKeys && k == 0) {
            w[2 * e] = code_pair<FMT, true, false>(x);
            w[2 * e + 1] = code_pair<FMT, true, true>(x);
          } else {
            w[2 * e] = scaled_pair<FMT, false>(x, s);
            w[2 * e + 1] = scaled_pair<FMT, true>(x, s);
          }
        }
        const int at = k == 0 ? k_chunk<HD>(r, c + q) : v_chunk<HD>(r, c + q);
        *reinterpret_cast<u32x4*>((k == 0 ? k_buf(i) : v_buf(i)) + r * kRowBytes + 16 * at) = w;
      }
    }
  };
  // Keys and values of tile i, just stored: e4m3 codes were scaled by their scale's exponent alone, and a scale of the caller's
  // that is no power of two has a factor left. One test per tile: a test with each conversion cost 4 % of a chunk.
  auto store_factors = [&](int i, const Held& hk, const Held& hv) {
    if constexpr (FMT == kFmtE4m3) {
      uint32_t bits = 0;
#pragma unroll
      for (int j = 0; j < kCLoads; ++j) bits |= (kRawKeys ? 0u : __float_as_uint(hk.scale[j])) | __float_as_uint(hv.scale[j]);
      if (__builtin_expect(__builtin_amdgcn_ballot_w64((bits & 0x807FFFFFu) != 0) == 0, 1)) return;
#pragma unroll
      for (int k = kRawKeys ? 1 : 0; k < 2; ++k)
#pragma unroll
        for (int j = 0; j < kCLoads; ++j) {
          const Held& h = k == 0 ? hk : hv;
          const int r = wave * kTr + kCrl * j + lane / kCpr, c = 2 * (lane % kCpr);
          const uint32_t s = __float_as_uint(h.scale[j]);
          const float f = (s & 0x7F800000u) ? __uint_as_float((s & 0x807FFFFFu) | 0x3F800000u) : 0.0f;  // 0: below 2^-126
#pragma unroll 1
          for (int x = 0; x < 8; ++x) {  // word by word, this lane's own: more at once spills at heads of 64
            const int at = k == 0 ? k_chunk<HD>(r, c + x / 4) : v_chunk<HD>(r, c + x / 4);
            uint32_t* const p = reinterpret_cast<uint32_t*>((k == 0 ? k_buf(i) : v_buf(i)) + r * kRowBytes + 16 * at) + x % 4;
            *p = pack_bf16(__uint_as_float(*p << 16) * f, __uint_as_float(*p & 0xFFFF0000u) * f);
          }
        }
    }
  };

  // Per-lane LDS addresses of V: key 4 half + (lane % 16) / 4, dims 16 ((lane / 16) % 2) + 4 (lane % 4) of a block.
  const int vkey = 4 * half + ((lane & 15) >> 2);
  const int vc = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
  const int v_off = vkey * kRowBytes + 8 * (lane & 1);

  struct Scores {
    f32x16 s[2];
  };
  auto scores = [&](auto nb, Scores& sc, int i) {
    constexpr int NB = decltype(nb)::value;
    const uint8_t* kt = k_buf(i);
#pragma unroll
    for (int kb = 0; kb < NB; ++kb) {
#pragma unroll
      for (int v = 0; v < 16; ++v) sc.s[kb][v] = 0.0f;
#pragma unroll
      for (int m = 0; m < kS; ++m) {
        const u32x4 kf = *reinterpret_cast<const u32x4*>(kt + (32 * kb + col) * kRowBytes + 16 * k_chunk<HD>(col, 2 * m + half));
        sc.s[kb] = Op<F16 || kRawKeys>::mfma(kf, qf[m], sc.s[kb]);
      }
    }
  };
  u32x4 pf[KP][4];
  auto probabilities = [&](auto nb, const Scores& sc) {
    constexpr int NB = decltype(nb)::value;
#pragma unroll
    for (int i = 0; i < 2 * NB; ++i) {
      float p[8];
#pragma unroll
      for (int v = 0; v < 8; ++v) p[v] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc.s[i / 2][8 * (i % 2) + v], c2, -mc));
      // The sum adds the probabilities as rounded (KP = 2: to 16 bits), so that a row's weights add up to one.
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t hi = Op<F16>::pack(p[2 * e], p[2 * e + 1]);
        pf[0][i][e] = hi;
        l_run = Op<F16>::add_pair(hi, l_run);
        if constexpr (KP == 2) {
          const uint32_t lo = Op<F16>::pack(p[2 * e] - __uint_as_float(hi << 16), p[2 * e + 1] - __uint_as_float(hi & 0xFFFF0000u));
          pf[1][i][e] = lo;
          l_run = Op<F16>::add_pair(lo, l_run);
        }
      }
    }
  };
  // Tile i: its scores, their softmax, and its part of the output.
  // Its first NB blocks of 32 keys: the others are behind all of the wave's rows.
  auto step = [&](auto nb, int i, uint64_t mask) {
    constexpr int NB = decltype(nb)::value;
    Scores sc;
    scores(nb, sc, i);
    if constexpr (kRawKeys) {
#pragma unroll
      for (int kb = 0; kb < NB; ++kb)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const f32x4 s = *reinterpret_cast<const f32x4*>(k_scales + (i & 1) * kKeys + 32 * kb + 8 * q + 4 * half);
#pragma unroll
          for (int r = 0; r < 4; ++r) sc.s[kb][4 * q + r] *= s[r];
        }
    }
    const int t0 = i * kKeys;
    if constexpr (CAP) {
      if (a.softcap <= kShortCap) {
#pragma unroll
        for (int kb = 0; kb < NB; ++kb)
#pragma unroll
          for (int v = 0; v < 16; ++v) sc.s[kb][v] = short_cap(sc.s[kb][v] * cap_exp, a.softcap);
      } else {
#pragma unroll
        for (int kb = 0; kb < NB; ++kb)
#pragma unroll
          for (int v = 0; v < 16; ++v) sc.s[kb][v] = tanh_of(sc.s[kb][v] * cap_scale) * a.softcap;
      }
    }
    if (mask != ~uint64_t(0) || t0 + kKeys - 1 > first_pos) {
#pragma unroll
      for (int kb = 0; kb < NB; ++kb) {
        // Bit 8 q + r: key 8 q + 4 half + r of the block is a key at or before this row's token.
        const int room = q_pos - t0 - 32 * kb - 4 * half;
        const uint32_t bits = (uint32_t(mask >> (32 * kb)) >> (4 * half)) & (room >= 31 ? ~0u : room < 0 ? 0u : (2u << room) - 1u);
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          const uint32_t keep = uint32_t(int32_t(bits << (31 - (8 * (v / 4) + v % 4))) >> 31);
          sc.s[kb][v] = __uint_as_float((__float_as_uint(sc.s[kb][v]) & keep) | (__float_as_uint(neg_inf) & ~keep));
        }
      }
    }
    float top = neg_inf;
#pragma unroll
    for (int kb = 0; kb < NB; ++kb)
#pragma unroll
      for (int v = 0; v < 16; ++v) top = fmaxf(top, sc.s[kb][v]);
    const float m_new = fmaxf(m_run, other_half_max(top));
    if (__builtin_amdgcn_ballot_w64(m_new > m_run)) {
      const float mc_new = m_new == neg_inf ? 0.0f : m_new * c2;
      const float alpha = m_run == neg_inf ? 0.0f : __builtin_amdgcn_exp2f(mc - mc_new);
      m_run = m_new;
      mc = mc_new;
      if (i > first_tile) {
        l_run *= alpha;
#pragma unroll
        for (int d = 0; d < kD; ++d)
#pragma unroll
          for (int v = 0; v < 16; ++v) o[d][v] *= alpha;
      }
    }
    probabilities(nb, sc);
    const uint8_t* vt = v_buf(i);
#pragma unroll
    for (int j = 0; j < 2 * NB; ++j)
#pragma unroll
      for (int d = 0; d < kD; ++d) {
        // Keys 16 j + vkey and 8 further: both have vkey's low bits, so one swizzle.
        const uint8_t* p0 = vt + 16 * j * kRowBytes + v_off + 16 * v_chunk<HD>(vkey, 4 * d + vc);
        const u32x2 lo = read_transposed(p0), hi = read_transposed(p0 + 8 * kRowBytes);
        const u32x4 vf = {lo.x, lo.y, hi.x, hi.y};
#pragma unroll
        for (int p = 0; p < KP; ++p) o[d] = Op<F16>::mfma(vf, pf[p][j], o[d]);
      }
  };

  if (n_tiles > first_tile) {
    if constexpr (SRC == kSrcPacked) {
      fetch_packed(0, 0);
      fetch_packed(1, 0);
      fetch_query();
      wait_vmcnt<0>();
      load_query();
      auto arrived = [&]() {
        wait_vmcnt<0>();  // this wave's rows of the tile
        wait_lgkmcnt0();  // its reads of the buffers that are refilled next
        __builtin_amdgcn_s_barrier();
      };
      const int whole = a.t_end % kKeys != 0 && a.t_end % kKeys <= 32 ? n_tiles - 1 : n_tiles;
      for (int i = 0; i < whole; ++i) {
        arrived();
        if (i + 1 < n_tiles) {
          fetch_packed(0, i + 1);
          fetch_packed(1, i + 1);
        }
        if (i * kKeys <= wave_last) step(Blocks<2>{}, i, ~uint64_t(0));
      }
      if (whole < n_tiles) {
        arrived();
        if (whole * kKeys <= wave_last) step(Blocks<1>{}, whole, ~uint64_t(0));
      }
    } else {
      Look look = look_at(first_tile);
      Place place = place_of(look, entry_of(first_tile, look));
      advance(look);
      int32_t entry = entry_of(first_tile + 1, look);
      Held hk = fetch_codes(0, place), hv = fetch_codes(1, place);
      fetch_query();
      store_codes(0, first_tile, hk, place.mask);
      store_codes(1, first_tile, hv, place.mask);
      store_factors(first_tile, hk, hv);
      wait_vmcnt<0>();
      load_query();
      for (int i = first_tile; i < n_tiles; ++i) {
        wait_lgkmcnt0();  // its stores of tile i, and its reads of the buffers that are refilled next
        __builtin_amdgcn_s_barrier();
        const uint64_t mask = place.mask;
        if (i + 1 < n_tiles) {
          place = place_of(look, entry);
          hk = fetch_codes(0, place);
          hv = fetch_codes(1, place);
          advance(look);
          entry = entry_of(i + 2, look);
        }
        if (i * kKeys <= wave_last) step(Blocks<2>{}, i, mask);
        if (i + 1 < n_tiles) {
          store_codes(0, i + 1, hk, place.mask);
          store_codes(1, i + 1, hv, place.mask);
          store_factors(i + 1, hk, hv);
        }
      }
    }
  }

  // ---- rows with anything that is not finite: once more, key by key, masked keys left out ----
  auto again = [&](uint64_t lanes) {
    if (lanes) {
      wait_vmcnt<0>();  // the rows' own stores
      uint32_t bad = uint32_t(lanes) | uint32_t(lanes >> 32);
      constexpr int kE = HD / 64;  // dims per lane
      for (; bad; bad &= bad - 1) {
        const int row = wrow + __builtin_ctz(bad);
        const int t_row = tok_of(row), g = row - t_row * a.group;
        const int pos = a.base + t_row;
        const uint16_t* q = static_cast<const uint16_t*>(a.query) + t_row * a.q_tok_stride + g * a.q_head_stride;
        auto element = [&](int k, int t, int d, bool& key) -> float {  // dim d of key (value) t
          if constexpr (SRC == kSrcPacked) {
            const uint16_t x = k == 0 ? a.key[t * a.k_tok_stride + d] : a.value[t * a.v_tok_stride + d];
            return F16 ? f16_to_f32(x) : bf16_to_f32(x);
          } else {
            const uint32_t bi = uint32_t(t) / a.block_size;
            const int32_t entry = bi < a.ldb ? a.table[bi] : -1;
            key = key && entry >= 0 && uint32_t(entry) < a.num_blocks;
            const int64_t bl = (key ? int64_t(entry) : 0) * a.kv_heads + a.kvh;
            return code_to_f32<FMT>(a.codes[k][(bl * a.block_size + uint32_t(t) % a.block_size) * HD + d], 0) * a.scales[k][bl];
          }
        };
        float m = neg_inf, sum = 0.0f, acc[kE] = {};
        for (int t0 = a.t_begin; t0 <= pos && t0 < a.t_end; t0 += 64) {
          const int t = t0 + lane;
          bool key = t <= pos && t < a.t_end;
          float dot = 0.0f;
          for (int d = 0; d < HD; ++d) {
            const float x = QF16 ? f16_to_f32(q[d]) : bf16_to_f32(q[d]);
            dot = __builtin_fmaf(x, element(0, key ? t : 0, d, key), dot);
          }
          float sc = dot * a.scale;
          if (CAP) sc = tanhf(sc / a.softcap) * a.softcap;
          sc = key ? sc * kLog2e : neg_inf;
          float top = sc;
#pragma unroll
          for (int off = 32; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, 64));
          const float m_new = fmaxf(m, top), ref = m_new == neg_inf ? 0.0f : m_new;
          const float alpha = m == neg_inf ? 0.0f : __builtin_amdgcn_exp2f(m - ref);
          m = m_new;
          const float p = key ? __builtin_amdgcn_exp2f(sc - ref) : 0.0f;
          sum *= alpha;
#pragma unroll
          for (int e = 0; e < kE; ++e) acc[e] *= alpha;
          uint64_t keys = __builtin_amdgcn_ballot_w64(key);
          for (; keys; keys &= keys - 1) {
            const int from = __builtin_ctzll(keys);
            const float pt = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(p), from));
            sum += pt;
            bool yes = true;
#pragma unroll
            for (int e = 0; e < kE; ++e) acc[e] = __builtin_fmaf(pt, element(1, t0 + from, kE * lane + e, yes), acc[e]);
          }
        }
        const bool no = SRC == kSrcPacked ? sum == 0.0f : !(sum > 0.0f);
        if constexpr (SRC == kSrcCodes) {
          if (a.part_out) {
#pragma unroll
            for (int e = 0; e < kE; ++e) a.part_out[int64_t(row) * HD + kE * lane + e] = no ? 0.0f : acc[e] / sum;
            if (lane == 0) a.part_lse[row] = sum == 0.0f ? neg_inf : m + __builtin_amdgcn_logf(sum);
            continue;
          }
        }
        uint16_t* dst = static_cast<uint16_t*>(a.out) + t_row * a.o_tok_stride + g * a.o_head_stride + kE * lane;
#pragma unroll
        for (int e = 0; e < kE; ++e) {
          const float v = no ? 0.0f : acc[e] / sum;
          dst[e] = QF16 ? f32_to_f16_rne(v) : f32_to_bf16_rne(v);
        }
      }
    }
  };

  if constexpr (SRC == kSrcCodes) {
    if (a.part_out) {
      // ---- a part of the keys: fp32 rows and their log-sum-exps, for the merge kernel ----
      const float l = other_half_sum(l_run);
      const float inv = 1.0f / l;
      bool bad_value = false;
      float* const dst = a.part_out + int64_t(own_row) * HD + 4 * half;
#pragma unroll
      for (int d = 0; d < kD; ++d)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          f32x4 v;
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            v[r] = l > 0.0f ? o[d][4 * q + r] * inv : 0.0f;
            bad_value |= !(__builtin_fabsf(v[r]) < __int_as_float(0x7F800000));
          }
          if (row_ok) *reinterpret_cast<f32x4*>(dst + 32 * d + 8 * q) = v;
        }
      if (row_ok && half == 0) a.part_lse[own_row] = l == 0.0f ? neg_inf : mc + __builtin_amdgcn_logf(l);  // NaN stays
      again(__builtin_amdgcn_ballot_w64(bad_value && row_ok));
      return;
    }
  }

  // ---- output: row col, dims 32 d + 8 q + 4 half + r, through LDS so that the stores are whole rows ----
  wait_lgkmcnt0();
  __builtin_amdgcn_s_barrier();  // every wave is past its last tile
  uint8_t* const stage = lds + wave * 32 * kRowBytes;
  {
    const float l = other_half_sum(l_run);
    // Zeros without keys; over the cache also for a sum that is no number (as the torch sequence's nan_to_num gives).
    const bool none = SRC == kSrcPacked ? l == 0.0f : !(l > 0.0f);
    const float inv = 1.0f / l;
    if (__builtin_amdgcn_ballot_w64(none))
#pragma unroll
      for (int d = 0; d < kD; ++d)
#pragma unroll
        for (int v = 0; v < 16; ++v) o[d][v] = none ? 0.0f : o[d][v];
    const float scale = none ? 1.0f : inv;
    float bad[2] = {0.0f, 0.0f};  // 0 x a number is 0, 0 x anything else is not
#pragma unroll
    for (int d = 0; d < kD; ++d)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        float v[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          v[r] = o[d][4 * q + r] * scale;
          bad[r % 2] = __builtin_fmaf(v[r], 0.0f, bad[r % 2]);
        }
        *reinterpret_cast<u32x2*>(stage + col * kRowBytes + 16 * k_chunk<HD>(col, 4 * d + q) + 8 * half) =
            u32x2{Op<QF16>::pack(v[0], v[1]), Op<QF16>::pack(v[2], v[3])};
      }
    wait_lgkmcnt0();  // the wave's own rows: no barrier
    char* const out = static_cast<char*>(a.out) + a.row0_tok * a.o_tok_stride * 2;
#pragma unroll
    for (int i = 0; i < 32 / kRpl; ++i) {
      const int r = kRpl * i + lane / kCh, c = lane % kCh;
      if (wrow + r >= a.rows) continue;
      const u32x4 w = *reinterpret_cast<const u32x4*>(stage + r * kRowBytes + 16 * k_chunk<HD>(r, c));
      // Non-temporal: 128 prompts of 128 84 -> 68 us.
      __builtin_nontemporal_store(w, reinterpret_cast<u32x4*>(out + (row_offset(r, a.o_tok_stride, a.o_head_stride) + 16 * c)));
    }
    const bool bad_value = bad[0] != 0.0f || bad[1] != 0.0f;
    again(__builtin_amdgcn_ballot_w64(bad_value && row_ok));
  }
}

}  // namespace tile
}  // namespace llmopt
