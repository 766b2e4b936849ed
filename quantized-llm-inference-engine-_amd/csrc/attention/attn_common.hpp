// Shared by the kernels of the 8-bit KV cache and of packed prompts: argument blocks, the code formats and
// their exact conversions to MFMA operands.
//
// Cache of one layer (llmopt_kvq.h): codes [num_blocks, kv_heads, block_size, head_dim], one byte each, and one
// fp32 scale per (block, KV head), as written a power of two (0: nothing but zeros; NaN: something that was not finite
// was written). A block of one head is one contiguous run of bytes: 2 KB at 16 tokens of 128.
//
// int8 codes (at most 8 significant bits) and e4m3 codes (4) are exact bf16 and fp16 numbers, so the operands of
// the products are the codes themselves; a key's scale multiplies its scores, a value's scale its probability, in
// fp32. A power of two commutes with every rounding to bf16 (both have 8 exponent bits), so this gives what
// dequantized operands would; another scale of the caller's rounds a value's product on its own.
#pragma once

#include "../qcommon.hpp"

namespace llmopt {

enum : int { kFmtInt8 = 0, kFmtE4m3 = 1 };

typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));

struct KvqCache {
  uint8_t* codes[2];  // keys, values
  float* scales[2];
  int64_t num_blocks, block_size, kv_heads, head_dim;
  const int32_t* block_ids;  // [num_seqs, ldb]
  int64_t ldb;
};

struct KvqWriteArgs {
  KvqCache c;
  const int32_t* offsets;     // [num_seqs] position of each sequence's first new token
  const int32_t* cu_seqlens;  // packed rows: [num_seqs + 1], sequence s is rows cu[s] .. cu[s + 1] - 1; null: uniform
  const int32_t* query_lens;  // uniform rows: tokens of each sequence that count; null: all q_len
  const void* src[2];         // element (s, j, h, d) at s * seq + j * tok + h * head + d; packed rows have no s
  int64_t seq_stride[2], tok_stride[2], head_stride[2];
  int64_t num_seqs, q_len, total_tokens;
  int64_t units;         // (sequence, block) pairs that the grid covers
  int64_t units_per_seq;  // uniform rows
};

struct KvqAttnArgs {
  KvqCache c;
  const void* query;  // element (s, h, j, d) at s * q_seq + h * q_head + j * q_tok + d
  int64_t q_seq_stride, q_head_stride, q_tok_stride;
  void* out;  // of the query's type
  int64_t o_seq_stride, o_head_stride, o_tok_stride;
  const int32_t* context_lens;  // [num_seqs]
  int64_t num_seqs, num_heads, q_len;
  int group;          // query heads per KV head
  float scale, softcap;
  int q_vec;          // query rows 16-byte aligned
  // splits of tiles_per_split 32-token tiles (the chunk kernel: an even number); partial results when splits > 1
  int splits, waves;
  int64_t tiles_per_split;
  float* part_out;  // [splits, num_seqs, kv_heads, group * q_len, head_dim], each normalized
  float* part_lse;  // [splits, num_seqs, kv_heads, group * q_len], powers of two
};

struct PackedAttnArgs {
  const void* query;  // [total, heads, d] rows of q_tok_stride and heads of q_head_stride elements; k, v, out likewise
  const void* key;
  const void* value;
  void* out;
  int64_t q_tok_stride, q_head_stride, k_tok_stride, k_head_stride, v_tok_stride, v_head_stride;
  int64_t o_tok_stride, o_head_stride;
  const int32_t* cu_seqlens;  // [num_seqs + 1]
  int64_t num_seqs, total_tokens, num_heads, kv_heads;
  int group;
  float scale, softcap;
  int zero_tail;  // rows behind the last sequence: 1 zeros, 0 left as they are
  int64_t blocks;  // row blocks that the grid covers, per KV head
  int64_t tail_blocks;  // further blocks that clear the tail
};

hipError_t launch_kvq_write(const KvqWriteArgs& a, int fmt, int src_dtype, bool vec, hipStream_t stream);
hipError_t launch_kvq_decode(const KvqAttnArgs& a, int fmt, int q_dtype, hipStream_t stream);
hipError_t launch_kvq_chunk(const KvqAttnArgs& a, int fmt, int q_dtype, hipStream_t stream);
// Merges the parts of a.splits > 1 splits into a.out.
hipError_t launch_kvq_merge(const KvqAttnArgs& a, int q_dtype, hipStream_t stream);
hipError_t launch_packed_attention(const PackedAttnArgs& a, int dtype, int64_t head_dim, hipStream_t stream);

// ---- conversions ---------------------------------------------------------------------------------

template <int FMT>
__device__ __forceinline__ float code_to_f32(uint32_t word, int byte) {
  if constexpr (FMT == kFmtInt8) {
    return float(int8_t(word >> (8 * byte)));
  } else {
    switch (byte) {
      case 0: return __builtin_amdgcn_cvt_f32_fp8(int(word), 0);
      case 1: return __builtin_amdgcn_cvt_f32_fp8(int(word), 1);
      case 2: return __builtin_amdgcn_cvt_f32_fp8(int(word), 2);
      default: return __builtin_amdgcn_cvt_f32_fp8(int(word), 3);
    }
  }
}

// Four numbers as codes, ties to even; int8: |v| <= 128, e4m3: |v| <= 448.
template <int FMT>
__device__ __forceinline__ uint32_t f32_to_codes(float a, float b, float c, float d) {
  if constexpr (FMT == kFmtInt8) {
    const uint32_t x = uint32_t(int(rintf(a))) & 0xFFu, y = uint32_t(int(rintf(b))) & 0xFFu;
    const uint32_t z = uint32_t(int(rintf(c))) & 0xFFu, w = uint32_t(int(rintf(d)));
    return x | (y << 8) | (z << 16) | (w << 24);
  } else {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true));
  }
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const f32x2 v = {lo, hi};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2_t));
}

// Bytes 2 HI and 2 HI + 1 of a word as a pair of 16-bit numbers, both conversions exact.
template <int FMT, bool F16, bool HI>
__device__ __forceinline__ uint32_t code_pair(uint32_t w) {
  if constexpr (FMT == kFmtE4m3) {
    if constexpr (F16)
      return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, HI));
    else
      return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, HI));
  } else {
    const float a = float(int8_t(w >> (HI ? 16 : 0))), b = float(int8_t(w >> (HI ? 24 : 8)));
    if constexpr (F16)
      return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(a, b));
    else
      return pack_bf16(a, b);
  }
}

// Bytes 2 HI and 2 HI + 1 of a word times their scale as a bf16 pair, exactly for a power of two (and a product that bf16
// holds). The e4m3 conversion takes the scale's exponent with it and nothing else (NaN gives NaN, and 0, whose codes are
// zeros, 2^-127): the caller multiplies by what another scale has left.
template <int FMT, bool HI>
__device__ __forceinline__ uint32_t scaled_pair(uint32_t w, float scale) {
  if constexpr (FMT == kFmtE4m3)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, HI));
  else
    return pack_bf16(float(int8_t(w >> (HI ? 16 : 0))) * scale, float(int8_t(w >> (HI ? 24 : 8))) * scale);
}

// Eight codes in order as one MFMA operand.
template <int FMT, bool F16>
__device__ __forceinline__ u32x4 code_operand(uint32_t lo, uint32_t hi) {
  return u32x4{code_pair<FMT, F16, false>(lo), code_pair<FMT, F16, true>(lo), code_pair<FMT, F16, false>(hi),
               code_pair<FMT, F16, true>(hi)};
}

// Byte i of `a` and of `b` as a bf16 pair, for i = 0 .. 3.
template <int FMT>
__device__ __forceinline__ void transpose_pairs(uint32_t a, uint32_t b, uint32_t out[4]) {
  if constexpr (FMT == kFmtE4m3) {
    const uint32_t lo = __builtin_amdgcn_perm(b, a, 0x05010400u), hi = __builtin_amdgcn_perm(b, a, 0x07030602u);
    out[0] = code_pair<FMT, false, false>(lo);
    out[1] = code_pair<FMT, false, true>(lo);
    out[2] = code_pair<FMT, false, false>(hi);
    out[3] = code_pair<FMT, false, true>(hi);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = pack_bf16(float(int8_t(a >> (8 * i))), float(int8_t(b >> (8 * i))));
  }
}

// v of the lanes l and l ^ 32 (or l ^ 16), combined by fmaxf or +, in every lane.
__device__ __forceinline__ float max_across_rows(float v) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_across_rows(float v) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// The packed sequence that owns grid unit `unit`, found by all 64 lanes of a wave. Sequence i's units begin at
// start(cu[i], i), strictly increasing; cu_seqlens is read within [0, total]. Each round asks 64 sequences at even distances
// and keeps one gap; the last round's lanes hold what the caller needs next (the sequence's rows, and its entry of
// `more`, if given), so that up to 64 sequences cost one round trip to memory.
struct Packed {
  int64_t s;           // the last sequence whose units begin at or before `unit` (0 if none does)
  int32_t first, end;  // its rows
  int32_t more;
};
template <class F>
__device__ __forceinline__ Packed find_packed(const int32_t* cu_seqlens, int64_t count, int64_t total, int64_t unit,
                                              const int32_t* more, F start) {
  const int lane = threadIdx.x & 63;
  auto clamped = [&](int32_t v) -> int32_t { return v < 0 ? 0 : v > total ? int32_t(total) : v; };
  int64_t lo = 0, n = count;  // the answer is in [lo, lo + n)
  for (;;) {
    const int64_t step = (n + 63) / 64;
    const bool in = lane * step < n;
    const int64_t i = lo + (in ? lane * step : 0);
    const int32_t first = clamped(cu_seqlens[i]), end = clamped(cu_seqlens[i + 1]);
    const int32_t extra = more ? more[i] : 0;
    const uint64_t votes = __builtin_amdgcn_ballot_w64(in && start(int64_t(first), i) <= unit);
    const int last = votes ? 63 - __builtin_clzll(votes) : 0;
    lo += last * step;
    if (step == 1)
      return Packed{lo, __builtin_amdgcn_readlane(first, last), __builtin_amdgcn_readlane(end, last),
                    __builtin_amdgcn_readlane(extra, last)};
    const int64_t left = n - last * step;
    n = left < step ? left : step;
  }
}

// Soft cap, cap tanh(x), as cap - 2 cap / (1 + 2^y) with y = 2 x log2(e): off by up to 2^-21 of the cap. Taken for 16-bit queries
// up to kShortCap, where that is 3e-5 in a score and so 2^-15 of a probability, a sixteenth of what an fp16 output is rounded
// by (2^-11), also where two pieces hold 16 bits of the probability. 4 prompts of 2048 in bf16 208 us, with tanh_of 265, with
// the library's tanhf 300; chunks of 4 x 512 tokens over int8 codes in fp16 218 and 270, tanhf spills.
constexpr float kShortCap = 64.0f;
__device__ __forceinline__ float short_cap(float y, float cap) {
  return __builtin_fmaf(-2.0f * cap, __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(y)), cap);
}

// tanh within 2^-21 of its value: its series up to x^9 below 0.3 (the next term is 5e-8 of it), else (1 - t) / (1 + t) with
// t = e^(-2 |x|), of which 1 - t is off by 2^-22 at 0.3 and by less above. A capped score is then off by 2^-21 of itself: 2^-15
// of a probability at a score of 64, more at larger ones, as the product's own rounding (2^-24 per term).
__device__ __forceinline__ float tanh_of(float x) {
  const float x2 = x * x;
  const float near = x * __builtin_fmaf(x2, __builtin_fmaf(x2, __builtin_fmaf(x2, __builtin_fmaf(x2, 62.0f / 2835, -17.0f / 315), 2.0f / 15), -1.0f / 3), 1.0f);
  const float t = __builtin_amdgcn_exp2f(__builtin_fabsf(x) * (-2.0f * 1.44269504088896340736f));
  const float far = (1.0f - t) * __builtin_amdgcn_rcpf(1.0f + t);
  return __builtin_fabsf(x) < 0.3f ? near : __builtin_copysignf(far, x);
}

}  // namespace llmopt
