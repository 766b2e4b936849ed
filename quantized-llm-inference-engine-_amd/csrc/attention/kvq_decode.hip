// Attention over the 8-bit KV cache, read in place from the block table: few query rows per KV head (a decode
// step's one token, or some).
//
//   out = softmax(scale q K^T [, soft-capped]) V over the keys t <= ctx - q_len + j of query token j, t < ctx, whose
//   block id names a block; the query heads h of KV head h / group share its keys.
//
// A workgroup of W waves owns (context split, KV head, 16 query rows, sequence); the rows of a KV head are its
// group x q_len (token-major). Its 32-token tiles are dealt to the waves in turn. Per tile and wave:
//   * K: lane (col, kb) = (l % 16, l / 16) loads 16 contiguous bytes (two for heads of 128) of tokens col and
//     16 + col, bytes 16 kb + 64 j of the row: two 8-dim operands of v_mfma_f32_16x16x32 each. The query's operands
//     hold the same dims, and a dot product does not mind their order;
//   * the scores of tokens 4 kb + r and 16 + 4 kb + r for row col arrive in the lane, times the block's scale;
//     online softmax in fp32, in powers of two;
//   * V: the lane loads HD / 16 contiguous bytes of those eight tokens, dims (HD / 16) col ..: byte i of the eight is
//     the A operand of MFMA i (v_mfma_f32_16x16x32: 16 dims x 32 tokens), and the eight probabilities, times
//     the block's scale, are its B operand as they lie: nothing crosses lanes.
// Two tiles of codes are in flight in registers while one is computed. The block ids and scales of up to 32 tiles
// are gathered beforehand, one 16-token half per lane, where 16 divides the block size (UNI: a half lies in one
// block, whose address is then scalar); else per token and tile.
// The waves merge in LDS; with several splits each workgroup writes its normalized part and log-sum-exp, and a
// second kernel merges them (2.3 us; first parts and log-sum-exps on their way before the length is known: 0.5 less).
//
// Bound by HBM at large batches (64 sequences of up to 8192, int8: 811 MB in 153 us, 5.3 TB/s, what a large copy
// reaches), by the chain of loads (length, table, codes, next codes) at small ones: 32 sequences of up to 640 in e4m3 10.8 us (32 MB;
// 24 with up to 4000 tokens and heads of 64 in fp16 17.9, one of 641 8.5 with its merge, in a graph). Sixteen waves
// per workgroup spill; one tile in flight, non-temporal loads and non-temporal queries measured level or slower.
//
// Roundings: bf16 queries: probabilities in bf16 (the sum adds them as rounded). fp16 queries: keys as fp16 operands,
// the probability in two bf16 pieces (16 significant bits). fp32 queries: the query in three bf16 pieces (exact),
// the probability in two. Everything else is fp32.
#include "attn_common.hpp"

namespace llmopt {
namespace {

typedef short s16x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ f32x4 mfma_bf16(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
                                                 0);
}
__device__ __forceinline__ f32x4 mfma_f16(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

constexpr float kLog2e = 1.44269504088896340736f;

template <int QT>
struct Pieces {
  static constexpr int kQ = QT == kDtF32 ? 3 : 1;   // bf16 (fp16) pieces of the query
  static constexpr int kP = QT == kDtBf16 ? 1 : 2;  // bf16 pieces of a probability
};

template <int QT, int FMT, int HD, int W, bool UNI>
__global__ void __launch_bounds__(64 * W) __attribute__((amdgpu_waves_per_eu(2))) kvq_decode_kernel(const KvqAttnArgs a) {
  constexpr int kJ = HD / 64;      // 16-byte loads of a key row per lane
  constexpr int kNm = 2 * kJ;      // score MFMAs per half (32 dims each)
  constexpr int kNv = HD / 16;     // P V MFMAs per tile, dims per lane and token
  constexpr int kVw = kNv / 4;     // words of V per lane and token
  constexpr int kQ = Pieces<QT>::kQ, kP = Pieces<QT>::kP;
  constexpr bool kF16 = QT == kDtF16;
  const int lane = threadIdx.x & 63;
  const int wave = W > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
  const int col = lane & 15, kb = lane >> 4;
  const uint32_t kv_heads = uint32_t(a.c.kv_heads);
  const int split = int(blockIdx.x);
  const int kvh = int(blockIdx.y % kv_heads), rb = int(blockIdx.y / kv_heads);
  const int64_t s = blockIdx.z;
  const int q_len = int(a.q_len), rows = a.group * q_len;
  const int row = 16 * rb + col;
  const bool row_ok = row < rows;
  const int tok = int(uint32_t(row) / uint32_t(a.group));
  const int last_tok = int(uint32_t(min(16 * rb + 15, rows - 1)) / uint32_t(a.group));
  const uint32_t bs = uint32_t(a.c.block_size), ldb = uint32_t(a.c.ldb), nblk = uint32_t(a.c.num_blocks);
  const int32_t* const table = a.c.block_ids + s * a.c.ldb;
  const int t_begin = int(split * a.tiles_per_split) * 32;
  auto tile_t0 = [&](int i) -> int { return t_begin + 32 * (wave + W * i); };
  // The first table entries do not wait for the context's length.
  int32_t first_entry = -1;
  if constexpr (UNI) {
    const uint32_t bi = uint32_t(tile_t0(lane / 2) + 16 * (lane & 1)) / bs;
    if (bi < ldb) first_entry = table[bi];
  }
  const int base = max(a.context_lens[s], 0) - q_len;  // position of query token 0
  const int q_pos = row_ok ? base + tok : -1;
  const int first_pos = base + int(uint32_t(16 * rb) / uint32_t(a.group));
  // The rows' keys: t < t_end, within the table (its width in tokens is below 2^31, checked on the host).
  const int t_end = max(0, min(base + last_tok + 1, int(ldb * bs)));
  const int n_all = min(int(a.tiles_per_split), (t_end - t_begin + 31) / 32);
  const int n_tiles = n_all > wave ? (n_all - wave + W - 1) / W : 0;
  if (a.splits > 1 && n_all <= 0) return;  // the merge does not read this part

  // ---- the query row col: dims 64 j + 16 kb + 8 h .. + 8 are operand 2 j + h ----
  u32x4 qf[kQ][kNm];
  {
    const int64_t q0 = s * a.q_seq_stride + (int64_t(kvh) * a.group + (row_ok ? row - tok * a.group : 0)) * a.q_head_stride +
                       int64_t(row_ok ? tok : 0) * a.q_tok_stride + 16 * kb;
#pragma unroll
    for (int m = 0; m < kNm; ++m) {
      const int d = 64 * (m / 2) + 8 * (m % 2);
      if constexpr (QT == kDtF32) {
        const float* q = static_cast<const float*>(a.query) + q0 + d;
        float x[8];
        if (a.q_vec) {
          const f32x4 v0 = *reinterpret_cast<const f32x4*>(q), v1 = *reinterpret_cast<const f32x4*>(q + 4);
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = v0[e], x[e + 4] = v1[e];
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] = q[e];
        }
        // x = hi + mid + lo, each remainder exact: 3 x 8 significant bits.
#pragma unroll
        for (int p = 0; p < 3; ++p) {
          u32x4 w;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            w[e] = pack_bf16(x[2 * e], x[2 * e + 1]);
            x[2 * e] -= __uint_as_float(w[e] << 16);
            x[2 * e + 1] -= __uint_as_float(w[e] & 0xFFFF0000u);
          }
          qf[p][m] = row_ok ? w : u32x4{0u, 0u, 0u, 0u};
        }
      } else {
        const uint16_t* q = static_cast<const uint16_t*>(a.query) + q0 + d;
        u32x4 w;
        if (a.q_vec) {
          w = *reinterpret_cast<const u32x4*>(q);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) w[e] = uint32_t(q[2 * e]) | (uint32_t(q[2 * e + 1]) << 16);
        }
        qf[0][m] = row_ok ? w : u32x4{0u, 0u, 0u, 0u};
      }
    }
  }

  const uint8_t* const kcodes = a.c.codes[0];
  const uint8_t* const vcodes = a.c.codes[1];
  // Row of token slot `slot` of `block` in the codes; below 2^31 (checked on the host).
  auto row_at = [&](uint32_t block, uint32_t slot) -> int32_t {
    return int32_t((block * kv_heads + uint32_t(kvh)) * bs + slot);
  };

  struct Tile {
    u32x4 k[2][kJ];       // tokens col and 16 + col
    uint32_t v[8][kVw];   // tokens 4 kb + r, then 16 + 4 kb + r
    uint32_t bits;        // which of the 32 tokens are keys
    float ks[UNI ? 2 : 8], vs[UNI ? 2 : 8];
  };

  const float neg_inf = -__int_as_float(0x7F800000);
  float m_run = neg_inf, l_run = 0.0f;  // running maximum of row col, and this lane's share of its sum
  f32x4 o[kNv];
#pragma unroll
  for (int i = 0; i < kNv; ++i) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  const bool capped = a.softcap > 0.0f;
  const float score_scale = capped ? a.scale / a.softcap : a.scale * kLog2e;
  const float cap2 = a.softcap * kLog2e;

  auto compute = [&](Tile& t, int t0) {
    // The codes as whole words here: without this the compiler keeps every byte in a register of its own across
    // the loop (300 registers instead of 150).
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < kJ; ++j) asm("" : "+v"(t.k[h][j]));
#pragma unroll
    for (int r = 0; r < 8; ++r)
#pragma unroll
      for (int w = 0; w < kVw; ++w) asm("" : "+v"(t.v[r][w]));
    f32x4 acc[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      acc[h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < kJ; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const u32x4 kf = code_operand<FMT, kF16>(t.k[h][j][2 * e], t.k[h][j][2 * e + 1]);
#pragma unroll
          for (int p = 0; p < kQ; ++p)
            acc[h] = kF16 ? mfma_f16(kf, qf[p][2 * j + e], acc[h]) : mfma_bf16(kf, qf[p][2 * j + e], acc[h]);
          __builtin_amdgcn_sched_barrier(0);  // one operand at a time: converted all at once they take 100 registers
        }
    }
    float sc[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) sc[r] = acc[r / 4][r % 4] * (score_scale * t.ks[UNI ? r / 4 : r]);
    if (capped) {
      if (QT != kDtF32 && a.softcap <= kShortCap) {
#pragma unroll
        for (int r = 0; r < 8; ++r) sc[r] = short_cap(sc[r] * (2.0f * kLog2e), cap2);
      } else {
#pragma unroll
        for (int r = 0; r < 8; ++r) sc[r] = tanhf(sc[r]) * cap2;
      }
    }
    const bool masked = t.bits != ~0u || t0 + 31 > first_pos;
    uint32_t keep = 0xFFu;
    if (masked) {
      keep = 0;
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        const int at = 16 * (r / 4) + 4 * kb + r % 4;
        const bool key = (t.bits >> at) & 1u;
        const bool seen = key && t0 + at <= q_pos;
        keep |= seen ? 1u << r : 0u;
        sc[r] = seen ? sc[r] : neg_inf;
        // A row that is no key may hold anything: its probability is 0, and so has to be its value.
#pragma unroll
        for (int w = 0; w < kVw; ++w) t.v[r][w] = key ? t.v[r][w] : 0u;
      }
    }
    float top = fmaxf(fmaxf(fmaxf(sc[0], sc[1]), fmaxf(sc[2], sc[3])), fmaxf(fmaxf(sc[4], sc[5]), fmaxf(sc[6], sc[7])));
    top = max_across_rows(top);
    if (__builtin_amdgcn_ballot_w64(top > m_run)) {
      const float m_new = fmaxf(m_run, top);
      const float alpha = m_run == neg_inf ? 0.0f : __builtin_amdgcn_exp2f(m_run - m_new);
      m_run = m_new;
      l_run *= alpha;
#pragma unroll
      for (int i = 0; i < kNv; ++i) o[i] *= alpha;
    }
    const float m_ref = m_run == neg_inf ? 0.0f : m_run;
    float p[8], pv[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      p[r] = __builtin_amdgcn_exp2f(sc[r] - m_ref);
      pv[r] = p[r] * t.vs[UNI ? r / 4 : r];
    }
    if (masked) {
#pragma unroll
      for (int r = 0; r < 8; ++r) pv[r] = (keep >> r) & 1u ? pv[r] : 0.0f;  // whatever the scale is
    }
    u32x4 pf[kP];
#pragma unroll
    for (int i = 0; i < 4; ++i) pf[0][i] = pack_bf16(pv[2 * i], pv[2 * i + 1]);
    if constexpr (kP == 2) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        pf[1][i] = pack_bf16(pv[2 * i] - __uint_as_float(pf[0][i] << 16),
                             pv[2 * i + 1] - __uint_as_float(pf[0][i] & 0xFFFF0000u));
      l_run += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
    } else {
      // The sum of the probabilities as rounded, so that a row's weights add up to one.
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        sum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, pack_bf16(p[2 * i], p[2 * i + 1])),
                                              __builtin_bit_cast(bf16x2_t, 0x3F803F80u), sum, false);
      l_run += sum;
    }
#pragma unroll
    for (int w = 0; w < kVw; ++w) {
      uint32_t pair[4][4];  // [tokens 2 i, 2 i + 1][dim]
#pragma unroll
      for (int i = 0; i < 4; ++i) transpose_pairs<FMT>(t.v[2 * i][w], t.v[2 * i + 1][w], pair[i]);
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        const u32x4 va = {pair[0][d], pair[1][d], pair[2][d], pair[3][d]};
#pragma unroll
        for (int q = 0; q < kP; ++q) o[4 * w + d] = mfma_bf16(va, pf[q], o[4 * w + d]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  auto load_k = [&](Tile& t, int half, const uint8_t* p) {
#pragma unroll
    for (int j = 0; j < kJ; ++j) t.k[half][j] = *reinterpret_cast<const u32x4*>(p + 64 * j);
  };
  auto load_v = [&](Tile& t, int r, const uint8_t* p) {
    if constexpr (kVw == 2) {
      const u32x2 w = *reinterpret_cast<const u32x2*>(p);
      t.v[r][0] = w.x, t.v[r][1] = w.y;
    } else {
      t.v[r][0] = *reinterpret_cast<const uint32_t*>(p);
    }
  };

  constexpr int kDepth = 2;  // tiles in flight behind the one that is computed
  Tile ring[kDepth];
  if constexpr (UNI) {
    const uint32_t k_lane = uint32_t(col * HD + 16 * kb), v_lane = uint32_t(4 * kb * HD + kNv * col);
    for (int g0 = 0; g0 < n_tiles; g0 += 32) {
      const int n = min(32, n_tiles - g0);
      // Lane l: half l % 2 of the group's tile l / 2.
      int32_t my_row = -1;
      float my_ks = 0.0f, my_vs = 0.0f;
      {
        const uint32_t t = uint32_t(tile_t0(g0 + lane / 2) + 16 * (lane & 1));
        const uint32_t bi = t / bs;
        if (g0 > 0) first_entry = bi < ldb ? table[bi] : -1;
        if (lane < 2 * n && int(t) < t_end) {
          const int32_t entry = first_entry;
          if (entry >= 0 && uint32_t(entry) < nblk) {
            my_row = row_at(uint32_t(entry), t - bi * bs);
            const int64_t at = int64_t(entry) * kv_heads + kvh;
            my_ks = a.c.scales[0][at];
            my_vs = a.c.scales[1][at];
          }
        }
      }
      auto fetch = [&](int i, Tile& t) {
        const int t0 = tile_t0(g0 + i);
        uint32_t bits = 0;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int32_t r = __builtin_amdgcn_readlane(my_row, 2 * i + h);
          const int64_t at = int64_t(r >= 0 ? r : 0) * HD;  // no key: some row of the cache
          load_k(t, h, kcodes + at + k_lane);
#pragma unroll
          for (int k = 0; k < 4; ++k) load_v(t, 4 * h + k, vcodes + at + v_lane + k * HD);
          t.ks[h] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(my_ks), 2 * i + h));
          t.vs[h] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(my_vs), 2 * i + h));
          const int room = t_end - t0 - 16 * h;  // tokens of this half before the end
          bits |= (r < 0 || room <= 0 ? 0u : room >= 16 ? 0xFFFFu : (1u << room) - 1u) << (16 * h);
        }
        t.bits = bits;
      };
#pragma unroll
      for (int u = 0; u < kDepth; ++u)
        if (u < n) fetch(u, ring[u]);
      for (int i = 0; i < n; i += kDepth) {
#pragma unroll
        for (int u = 0; u < kDepth; ++u)
          if (i + u < n) {
            compute(ring[u], tile_t0(g0 + i + u));
            if (i + u + kDepth < n) fetch(i + u + kDepth, ring[u]);
          }
      }
    }
  } else {
    auto fetch = [&](int i, Tile& t) {
      const uint32_t tt = uint32_t(tile_t0(i) + (lane & 31));
      const uint32_t bi = tt / bs;
      int32_t my_row = -1;
      float my_ks = 0.0f, my_vs = 0.0f;
      if (int(tt) < t_end) {
        const int32_t entry = table[bi];
        if (entry >= 0 && uint32_t(entry) < nblk) {
          my_row = row_at(uint32_t(entry), tt - bi * bs);
          const int64_t at = int64_t(entry) * kv_heads + kvh;
          my_ks = a.c.scales[0][at];
          my_vs = a.c.scales[1][at];
        }
      }
      t.bits = uint32_t(__builtin_amdgcn_ballot_w64(my_row >= 0));
      const int32_t r_own = my_row >= 0 ? my_row : 0;
#pragma unroll
      for (int h = 0; h < 2; ++h)
        load_k(t, h, kcodes + int64_t(__shfl(r_own, 16 * h + col, 64)) * HD + 16 * kb);
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        const int from = 16 * (r / 4) + 4 * kb + r % 4;
        load_v(t, r, vcodes + int64_t(__shfl(r_own, from, 64)) * HD + kNv * col);
        t.ks[UNI ? 0 : r] = __shfl(my_ks, from, 64);
        t.vs[UNI ? 0 : r] = __shfl(my_vs, from, 64);
      }
    };
#pragma unroll
    for (int u = 0; u < kDepth; ++u)
      if (u < n_tiles) fetch(u, ring[u]);
    for (int i = 0; i < n_tiles; i += kDepth) {
#pragma unroll
      for (int u = 0; u < kDepth; ++u)
        if (i + u < n_tiles) {
          compute(ring[u], tile_t0(i + u));
          if (i + u + kDepth < n_tiles) fetch(i + u + kDepth, ring[u]);
        }
    }
  }

  // ---- the waves' parts: lane (col, kb) holds row col, dims kNv (4 kb + r) + i ----
  l_run = sum_across_rows(l_run);
  extern __shared__ __align__(16) float merge_lds[];  // [W][16] maxima, sums; [W][rows][HD + 4]: launch_waves sizes it
  const int here = min(16, rows - 16 * rb);
  float(*const m_lds)[16] = reinterpret_cast<float(*)[16]>(merge_lds);
  float(*const l_lds)[16] = m_lds + W;
  float* const o_lds = merge_lds + 2 * W * 16;
  if (kb == 0) m_lds[wave][col] = m_run, l_lds[wave][col] = l_run;
  if (row_ok) {
    float* const at = o_lds + (wave * here + col) * (HD + 4);
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int i = 0; i < kNv; ++i) at[kNv * (4 * kb + r) + i] = o[i][r];
  }
  __syncthreads();
  for (int e = int(threadIdx.x); e < here * HD; e += 64 * W) {
    const int rr = e / HD, d = e % HD;
    float top = neg_inf;
#pragma unroll
    for (int w = 0; w < W; ++w) top = fmaxf(top, m_lds[w][rr]);
    float lsum = 0.0f, acc = 0.0f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float mw = m_lds[w][rr];
      const float f = mw == neg_inf ? 0.0f : __builtin_amdgcn_exp2f(mw - top);
      lsum = __builtin_fmaf(f, l_lds[w][rr], lsum);
      acc = __builtin_fmaf(f, o_lds[(w * here + rr) * (HD + 4) + d], acc);
    }
    // Zeros without keys, and for a sum that is no number (as the torch sequence's nan_to_num gives).
    const float val = lsum > 0.0f ? acc / lsum : 0.0f;
    const int r = 16 * rb + rr;
    if (a.splits == 1) {
      const int t = int(uint32_t(r) / uint32_t(a.group));
      const int64_t at = s * a.o_seq_stride + (int64_t(kvh) * a.group + (r - t * a.group)) * a.o_head_stride +
                         int64_t(t) * a.o_tok_stride + d;
      if constexpr (QT == kDtF32) static_cast<float*>(a.out)[at] = val;
      if constexpr (QT == kDtF16) static_cast<uint16_t*>(a.out)[at] = f32_to_f16_rne(val);
      if constexpr (QT == kDtBf16) static_cast<uint16_t*>(a.out)[at] = f32_to_bf16_rne(val);
    } else {
      const int64_t at = ((int64_t(split) * a.num_seqs + s) * kv_heads + kvh) * rows + r;
      a.part_out[at * HD + d] = val;
      if (d == 0) a.part_lse[at] = lsum == 0.0f ? neg_inf : top + __builtin_amdgcn_logf(lsum);  // NaN stays
    }
  }
}

// The splits of one (sequence, KV head, row), one wave: weights 2^(lse - max lse).
template <int QT, int HD>
__global__ void __launch_bounds__(256) kvq_merge_kernel(const KvqAttnArgs a) {
  constexpr int kD = HD / 64;
  const int lane = threadIdx.x & 63;
  const int rows = a.group * int(a.q_len);
  const uint32_t kv_heads = uint32_t(a.c.kv_heads);
  const int r = int(blockIdx.x) * 4 + int(threadIdx.x >> 6);
  const int64_t kvh = blockIdx.y, s = blockIdx.z;
  if (r >= rows) return;
  const float neg_inf = -__int_as_float(0x7F800000);
  const int64_t stride = a.num_seqs * int64_t(kv_heads) * rows;  // between two splits
  const float* const lse_at = a.part_lse + (s * kv_heads + kvh) * rows + r;
  const float* const part = a.part_out + ((s * kv_heads + kvh) * rows + r) * HD + kD * lane;
  // The log-sum-exps, a split per lane, and the first parts are on their way before the context's length, which says
  // how many there are, is known: parts past it were not written and are not used.
  constexpr int kAhead = 4;
  float ahead[kAhead][kD];
#pragma unroll
  for (int i = 0; i < kAhead; ++i)
#pragma unroll
    for (int d = 0; d < kD; ++d) ahead[i][d] = i < a.splits ? part[i * stride * HD + d] : 0.0f;
  float lse = lane < a.splits ? lse_at[lane * stride] : neg_inf;
  // The splits that the row's block of 16 ran.
  const int base = max(a.context_lens[s], 0) - int(a.q_len);
  const int last_tok = int(uint32_t(min((r & ~15) + 15, rows - 1)) / uint32_t(a.group));
  const int t_end = max(0, min(base + last_tok + 1, int(a.c.ldb * a.c.block_size)));
  const int span = int(a.tiles_per_split) * 32;
  const int n = min(a.splits, (t_end + span - 1) / span);
  lse = lane < n ? lse : neg_inf;
  float top = lse;
  for (int i = 64 + lane; i < n; i += 64) top = fmaxf(top, lse_at[i * stride]);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
  float acc[kD] = {}, sum = 0.0f;
  if (top != neg_inf) {
    auto weight = [&](float x) { return x == neg_inf ? 0.0f : __builtin_amdgcn_exp2f(x - top); };
    const float w_lane = weight(lse);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const float w = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w_lane), i));
      if (i < n) {
        sum += w;
#pragma unroll
        for (int d = 0; d < kD; ++d) acc[d] = __builtin_fmaf(w, ahead[i][d], acc[d]);
      }
    }
#pragma unroll 4
    for (int i = kAhead; i < n; ++i) {
      const float w = i < 64 ? __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w_lane), i & 63))
                             : weight(lse_at[i * stride]);
      sum += w;
#pragma unroll
      for (int d = 0; d < kD; ++d) acc[d] = __builtin_fmaf(w, part[i * stride * HD + d], acc[d]);
    }
  }
  const int tok = int(uint32_t(r) / uint32_t(a.group));
  const int64_t out = s * a.o_seq_stride + (kvh * a.group + (r - tok * a.group)) * a.o_head_stride +
                      int64_t(tok) * a.o_tok_stride + kD * lane;
#pragma unroll
  for (int d = 0; d < kD; ++d) {
    const float v = sum > 0.0f ? acc[d] / sum : 0.0f;
    if constexpr (QT == kDtF32) static_cast<float*>(a.out)[out + d] = v;
    if constexpr (QT == kDtF16) static_cast<uint16_t*>(a.out)[out + d] = f32_to_f16_rne(v);
    if constexpr (QT == kDtBf16) static_cast<uint16_t*>(a.out)[out + d] = f32_to_bf16_rne(v);
  }
}

template <int QT, int FMT, int HD, bool UNI>
hipError_t launch_waves(const KvqAttnArgs& a, hipStream_t stream) {
  const int64_t rows = a.group * a.q_len, blocks = (rows + 15) / 16;
  const dim3 grid(unsigned(a.splits), unsigned(a.c.kv_heads * blocks), unsigned(a.num_seqs));
  const size_t lds = size_t(a.waves) * (2 * 16 + size_t(rows < 16 ? rows : 16) * (HD + 4)) * sizeof(float);
  switch (a.waves) {
    case 4: hipLaunchKernelGGL((kvq_decode_kernel<QT, FMT, HD, 4, UNI>), grid, dim3(256), lds, stream, a); break;
    case 8: hipLaunchKernelGGL((kvq_decode_kernel<QT, FMT, HD, 8, UNI>), grid, dim3(512), lds, stream, a); break;
    default: return hipErrorInvalidValue;
  }
  if (a.splits > 1) return launch_kvq_merge(a, QT, stream);
  return hipGetLastError();
}

template <int QT, int FMT>
hipError_t launch_hd(const KvqAttnArgs& a, hipStream_t stream) {
  const bool uni = a.c.block_size % 16 == 0;
  if (a.c.head_dim == 128)
    return uni ? launch_waves<QT, FMT, 128, true>(a, stream) : launch_waves<QT, FMT, 128, false>(a, stream);
  return uni ? launch_waves<QT, FMT, 64, true>(a, stream) : launch_waves<QT, FMT, 64, false>(a, stream);
}

template <int QT>
hipError_t launch_fmt(const KvqAttnArgs& a, int fmt, hipStream_t stream) {
  return fmt == kFmtInt8 ? launch_hd<QT, kFmtInt8>(a, stream) : launch_hd<QT, kFmtE4m3>(a, stream);
}

template <int QT>
void launch_merge(const KvqAttnArgs& a, hipStream_t stream) {
  const int64_t rows = a.group * a.q_len;
  const dim3 grid(unsigned((rows + 3) / 4), unsigned(a.c.kv_heads), unsigned(a.num_seqs));
  if (a.c.head_dim == 128)
    hipLaunchKernelGGL((kvq_merge_kernel<QT, 128>), grid, dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL((kvq_merge_kernel<QT, 64>), grid, dim3(256), 0, stream, a);
}

}  // namespace

hipError_t launch_kvq_merge(const KvqAttnArgs& a, int q_dtype, hipStream_t stream) {
  switch (q_dtype) {
    case kDtF32: launch_merge<kDtF32>(a, stream); break;
    case kDtF16: launch_merge<kDtF16>(a, stream); break;
    default: launch_merge<kDtBf16>(a, stream); break;
  }
  return hipGetLastError();
}

hipError_t launch_kvq_decode(const KvqAttnArgs& a, int fmt, int q_dtype, hipStream_t stream) {
  if (a.num_seqs == 0 || a.q_len == 0) return hipSuccess;
  switch (q_dtype) {
    case kDtF32: return launch_fmt<kDtF32>(a, fmt, stream);
    case kDtF16: return launch_fmt<kDtF16>(a, fmt, stream);
    default: return launch_fmt<kDtBf16>(a, fmt, stream);
  }
}

}  // namespace llmopt
