// Quantizing writes into the 8-bit KV cache: a decode step's tokens, chunks, and packed prompts.
//
// One wave takes one (sequence, cache block, KV head, K or V): the new rows that fall into that block. It holds
// them in registers (blocks of more than 8 x 64 chunks of 8 numbers are read twice), takes their largest magnitude, fixes
// the scale and writes the codes. Bound by HBM (3 bytes per 16-bit number) and, one wave's work being 4 KB, by its chain of
// loads: lengths and offsets, then the rows and the table entry together. Measured (MI355X, bf16, 8 heads of 128, blocks of
// 16): 32 prompts of 1 - 1024 tokens 20.8 us (104 MB, 5.0 TB/s; 36 with the table before the rows and numbers held as fp32),
// one token of 256 sequences 5.5, of one sequence 4.2.
//   need  = 2^e, the smallest e >= -126 with amax <= top 2^e (top = 127 or 448), 0 for amax = 0, NaN for a row
//           that holds an infinity or a NaN
//   scale = need where the write holds the block's slot 0 (the block starts anew), else max(old, need)
//   code  = x / scale, ties to even (codes 0 for a NaN scale)
// and where the scale grew, the block's other slots are rounded to the new one. All of it is exact in fp32 but
// for the one rounding of each code: the scales are powers of two. Magnitudes are compared as their bits, so a
// NaN counts as the largest.
#include "attn_common.hpp"

namespace llmopt {
namespace {

constexpr int kWaves = 4;

template <int FMT>
__device__ __forceinline__ uint32_t scale_bits_for(uint32_t amax_bits) {
  if (amax_bits == 0) return 0u;
  if (amax_bits >= 0x7F800000u) return 0x7FC00000u;
  // amax = f 2^k with f in [1, 2): e = k - 6 (127 = 1.984375 2^6) or k - 8 (448 = 1.75 2^8), one more above top's f.
  constexpr int kShift = FMT == kFmtInt8 ? 6 : 8;
  constexpr uint32_t kFraction = FMT == kFmtInt8 ? 0x7E0000u : 0x600000u;
  const int e = int(amax_bits >> 23) - kShift + ((amax_bits & 0x7FFFFFu) > kFraction ? 1 : 0);  // biased
  return uint32_t(e < 1 ? 1 : e) << 23;
}

// A chunk as it lies in memory: eight numbers (16-byte aligned) or one.
template <int SRC, bool VEC>
struct Chunk;
template <>
struct Chunk<kDtF32, true> {
  f32x4 w[2];
  __device__ void load(const void* p, int64_t i) {
    w[0] = *reinterpret_cast<const f32x4*>(static_cast<const float*>(p) + i);
    w[1] = *reinterpret_cast<const f32x4*>(static_cast<const float*>(p) + i + 4);
  }
  __device__ void clear() { w[0] = w[1] = f32x4{0.f, 0.f, 0.f, 0.f}; }
  __device__ float get(int e) const { return w[e / 4][e % 4]; }
};
template <int SRC>
struct Chunk<SRC, true> {
  u32x4 w;
  __device__ void load(const void* p, int64_t i) { w = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(p) + i); }
  __device__ void clear() { w = u32x4{0u, 0u, 0u, 0u}; }
  __device__ float get(int e) const {
    const uint32_t x = w[e / 2];
    if constexpr (SRC == kDtF16) return f16_to_f32(uint16_t(e % 2 ? x >> 16 : x));
    return __uint_as_float(e % 2 ? x & 0xFFFF0000u : x << 16);
  }
};
template <int SRC>
struct Chunk<SRC, false> {
  float x;
  __device__ void load(const void* p, int64_t i) {
    if constexpr (SRC == kDtF32) x = static_cast<const float*>(p)[i];
    if constexpr (SRC == kDtF16) x = f16_to_f32(static_cast<const uint16_t*>(p)[i]);
    if constexpr (SRC == kDtBf16) x = bf16_to_f32(static_cast<const uint16_t*>(p)[i]);
  }
  __device__ void clear() { x = 0.0f; }
  __device__ float get(int) const { return x; }
};

// VEC: head_dim a multiple of 8 and every source row 16-byte aligned: chunks of 8 numbers, else single ones. A lane holds
// kKeep chunks in registers: 4 cover blocks of up to 2048 numbers (16 x 128) at 44 registers, 8 one twice as long at 68
// (write_32 27.5 us with 4, 29.4 with 8).
template <int SRC, int FMT, bool VEC, int kKeep>
__global__ void __launch_bounds__(64 * kWaves) kvq_write_kernel(const KvqWriteArgs a) {
  constexpr int E = VEC ? 8 : 1;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t kv_heads = uint32_t(a.c.kv_heads);
  const uint32_t groups = (2 * kv_heads + kWaves - 1) / kWaves;
  const uint32_t hs = blockIdx.x % groups * kWaves + uint32_t(wave);
  const uint32_t unit = blockIdx.x / groups;
  if (hs >= 2 * kv_heads) return;
  const int side = hs >= kv_heads;
  const int64_t h = side ? hs - kv_heads : hs;
  const int64_t bs = a.c.block_size, hd = a.c.head_dim;

  // ---- the unit's sequence, block and rows ----
  int64_t s, j, row0, len, off;  // block j of the sequence's new ones; their source row, count and position
  if (a.cu_seqlens) {
    // Sequence i's units start at floor(cu[i] / bs) + 2 i: room for the len / bs + 2 blocks it can touch.
    auto start = [&](int64_t at, int64_t i) -> int64_t { return uint32_t(at) / uint32_t(bs) + 2 * i; };
    const Packed p = find_packed(a.cu_seqlens, a.num_seqs, a.total_tokens, unit, a.offsets, start);
    s = p.s;
    j = unit - start(p.first, s);
    row0 = p.first;
    len = p.end - p.first;
    off = p.more;
  } else {
    s = unit / uint32_t(a.units_per_seq);
    j = unit - s * a.units_per_seq;
    row0 = 0;
    len = a.query_lens ? a.query_lens[s] : a.q_len;
    if (len > a.q_len) len = a.q_len;
    off = a.offsets[s];
  }
  if (off < 0 || j < 0) return;
  const int64_t first = uint32_t(off) / uint32_t(bs), jb = first + j;  // 32 bits: checked on the host
  const int64_t p0 = j == 0 ? off : jb * bs;
  const int64_t p1 = off + len < (jb + 1) * bs ? off + len : (jb + 1) * bs;
  if (p0 >= p1 || jb >= a.c.ldb) return;
  const int lo = int(p0 - jb * bs), hi = int(p1 - jb * bs);  // the new slots

  // ---- the new rows, on their way while the table is read ----
  const int64_t esize = SRC == kDtF32 ? 4 : 2;
  const int64_t src0 = (a.cu_seqlens ? row0 * a.tok_stride[side] : s * a.seq_stride[side]) +
                       (p0 - off) * a.tok_stride[side] + h * a.head_stride[side];
  const uint8_t* const src = static_cast<const uint8_t*>(a.src[side]) + src0 * esize;
  const int64_t tok_stride = a.tok_stride[side];
  const uint32_t parts = uint32_t(hd / E);
  const int shift = (parts & (parts - 1)) == 0 ? __builtin_ctz(parts) : -1;
  const uint32_t chunks = uint32_t(hi - lo) * parts;
  Chunk<SRC, VEC> x[kKeep];
  auto load = [&](uint32_t base) {
#pragma unroll
    for (int i = 0; i < kKeep; ++i) {
      const uint32_t c = base + 64 * i + lane;
      const uint32_t r = shift >= 0 ? c >> shift : c / parts, d = (c - r * parts) * E;
      if (c < chunks)
        x[i].load(src, r * tok_stride + d);
      else
        x[i].clear();
    }
  };
  load(0);

  // A sequence stops at its table row's first negative block.
  const int32_t* table = a.c.block_ids + s * a.c.ldb;
  int32_t entry = 0;
  for (int64_t i = first; i <= jb; i += 64) {
    entry = i + lane <= jb ? table[i + lane] : 0;
    if (__builtin_amdgcn_ballot_w64(entry < 0)) return;
  }
  const int64_t block = __builtin_amdgcn_readlane(entry, int(jb - first) & 63);
  if (block >= a.c.num_blocks) return;
  uint8_t* const codes = a.c.codes[side] + (block * kv_heads + h) * bs * hd;
  float* const scale_at = a.c.scales[side] + block * kv_heads + h;
  const uint32_t old_bits = lo > 0 ? __float_as_uint(*scale_at) & 0x7FFFFFFFu : 0u;

  // ---- their largest magnitude ----
  constexpr uint32_t kHeld = 64 * kKeep;
  uint32_t amax = 0;
  for (uint32_t base = 0; base < chunks; base += kHeld) {
    if (base > 0) load(base);
#pragma unroll
    for (int i = 0; i < kKeep; ++i)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const uint32_t m = __float_as_uint(x[i].get(e)) & 0x7FFFFFFFu;
        amax = m > amax ? m : amax;
      }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const uint32_t m = uint32_t(__shfl_xor(int(amax), o, 64));
    amax = m > amax ? m : amax;
  }
  const uint32_t need = scale_bits_for<FMT>(amax);
  const uint32_t bits = need > old_bits ? need : old_bits;
  const float scale = __uint_as_float(bits);
  const bool finite = bits < 0x7F800000u;
  const float inv = bits != 0 && finite ? 1.0f / scale : 0.0f;

  // ---- a grown scale: the block's other slots are rounded to it ----
  if (lo > 0 && finite && bits != old_bits) {
    const float ratio = __uint_as_float(old_bits) * inv;
    const uint32_t all = uint32_t(bs) * parts, skip0 = uint32_t(lo) * parts, skip1 = uint32_t(hi) * parts;
    for (uint32_t c = lane; c < all; c += 64) {
      if (c >= skip0 && c < skip1) continue;
      if constexpr (VEC) {
        u32x2* const at = reinterpret_cast<u32x2*>(codes + int64_t(c) * 8);
        u32x2 w = *at;
#pragma unroll
        for (int k = 0; k < 2; ++k)
          w[k] = f32_to_codes<FMT>(code_to_f32<FMT>(w[k], 0) * ratio, code_to_f32<FMT>(w[k], 1) * ratio,
                                   code_to_f32<FMT>(w[k], 2) * ratio, code_to_f32<FMT>(w[k], 3) * ratio);
        *at = w;
      } else {
        codes[c] = uint8_t(f32_to_codes<FMT>(code_to_f32<FMT>(codes[c], 0) * ratio, 0.f, 0.f, 0.f));
      }
    }
  }

  // ---- the new codes ----
  uint8_t* const dst = codes + int64_t(lo) * hd;
  for (uint32_t base = 0; base < chunks; base += kHeld) {
    if (chunks > kHeld) load(base);
#pragma unroll
    for (int i = 0; i < kKeep; ++i) {
      const uint32_t c = base + 64 * i + lane;
      if (c >= chunks) continue;
      float v[E];  // 0 under a NaN scale: what is not finite has no code
#pragma unroll
      for (int e = 0; e < E; ++e) v[e] = finite ? x[i].get(e) * inv : 0.0f;
      if constexpr (VEC)
        __builtin_nontemporal_store(
            u32x2{f32_to_codes<FMT>(v[0], v[1], v[2], v[3]), f32_to_codes<FMT>(v[4], v[5], v[6], v[7])},
            reinterpret_cast<u32x2*>(dst + int64_t(c) * 8));  // 32 prompts: 27.8 -> 23.1 us
      else
        dst[c] = uint8_t(f32_to_codes<FMT>(v[0], 0.f, 0.f, 0.f));
    }
  }
  if (lane == 0 && (lo == 0 || bits != old_bits)) *scale_at = scale;
}

template <int SRC, int FMT>
void launch_vec(const KvqWriteArgs& a, bool vec, dim3 grid, hipStream_t stream) {
  if (vec) {
    if (a.c.block_size * a.c.head_dim <= 64 * 4 * 8)
      hipLaunchKernelGGL((kvq_write_kernel<SRC, FMT, true, 4>), grid, dim3(64 * kWaves), 0, stream, a);
    else
      hipLaunchKernelGGL((kvq_write_kernel<SRC, FMT, true, 8>), grid, dim3(64 * kWaves), 0, stream, a);
  } else {
    hipLaunchKernelGGL((kvq_write_kernel<SRC, FMT, false, 8>), grid, dim3(64 * kWaves), 0, stream, a);
  }
}

template <int SRC>
void launch_fmt(const KvqWriteArgs& a, int fmt, bool vec, dim3 grid, hipStream_t stream) {
  if (fmt == kFmtInt8)
    launch_vec<SRC, kFmtInt8>(a, vec, grid, stream);
  else
    launch_vec<SRC, kFmtE4m3>(a, vec, grid, stream);
}

}  // namespace

hipError_t launch_kvq_write(const KvqWriteArgs& a, int fmt, int src_dtype, bool vec, hipStream_t stream) {
  const int64_t groups = (2 * a.c.kv_heads + kWaves - 1) / kWaves;
  const int64_t total = groups * a.units;
  if (total <= 0) return hipSuccess;
  if (total > 0x7FFFFFFF) return hipErrorInvalidValue;
  const dim3 grid{unsigned(total)};
  switch (src_dtype) {
    case kDtF32: launch_fmt<kDtF32>(a, fmt, vec, grid, stream); break;
    case kDtF16: launch_fmt<kDtF16>(a, fmt, vec, grid, stream); break;
    default: launch_fmt<kDtBf16>(a, fmt, vec, grid, stream); break;
  }
  return hipGetLastError();
}

}  // namespace llmopt
