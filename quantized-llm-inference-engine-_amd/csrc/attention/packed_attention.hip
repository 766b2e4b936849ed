// Causal attention over packed prompts (PackedAttention.forward): sequence s is rows cu_seqlens[s] .. cu_seqlens[s + 1]
// - 1 of query [total, heads, d] and key / value [total, kv_heads, d]; a token sees its sequence's tokens up to itself.
// The tile kernel of tile_attention.hpp over 16-bit rows (its times are there). Four workgroups per CU at heads of 64 (three with
// a soft cap), two of 128 (registers and LDS alike); the grid is sized by the rows, one block more per sequence, without reading cu_seqlens
// on the host, so a workgroup first finds its sequence by a search with one ballot per 64 of them.
#include "tile_attention.hpp"

namespace llmopt {
namespace {

using namespace tile;

template <bool F16, int HD, bool CAP>
__global__ void __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(HD == 128 ? 2 : CAP ? 3 : 4, HD == 128 ? 2 : CAP ? 3 : 4)))
    packed_attention_kernel(const PackedAttnArgs a) {
  __shared__ __align__(16) uint8_t lds[4 * kKeys * HD * 2];
  const uint32_t kv_heads = uint32_t(a.kv_heads);
  const uint32_t unit = blockIdx.x / kv_heads, kvh = blockIdx.x - unit * kv_heads;
  if (unit >= a.blocks) {
    auto cu = [&](int64_t i) -> int64_t {
      const int64_t v = a.cu_seqlens[i];
      return v < 0 ? 0 : v > a.total_tokens ? a.total_tokens : v;
    };
    // Rows in front of the first sequence (there are none in a proper call) and behind the last one: zeros.
    const int64_t lo = a.num_seqs > 0 ? cu(0) : a.total_tokens, hi = a.num_seqs > 0 ? cu(a.num_seqs) : a.total_tokens;
    const int64_t per_row = a.group * (HD / 8);
    for (int64_t i = (unit - a.blocks) * (64 * kWaves) + threadIdx.x; i < (lo + a.total_tokens - hi) * per_row;
         i += a.tail_blocks * (64 * kWaves)) {
      const int64_t r = i / per_row, x = i - r * per_row;
      const int64_t tok = r < lo ? r : hi + r - lo;
      uint16_t* dst = static_cast<uint16_t*>(a.out) + tok * a.o_tok_stride + (kvh * int64_t(a.group) + x / (HD / 8)) * a.o_head_stride;
      *reinterpret_cast<u32x4*>(dst + 8 * (x % (HD / 8))) = u32x4{0u, 0u, 0u, 0u};
    }
    return;
  }
  // Sequence i's row blocks start at floor(cu[i] group / kRows) + i: room for the ceil(len group / kRows) it has.
  auto start = [&](int64_t first, int64_t i) -> int64_t { return uint32_t(first) * uint32_t(a.group) / uint32_t(kRows) + i; };
  const Packed p = find_packed(a.cu_seqlens, a.num_seqs, a.total_tokens, int64_t(unit), nullptr, start);
  const int64_t first = p.first, len = p.end - p.first;
  const int64_t block = int64_t(unit) - start(first, p.s), count = (len * a.group + kRows - 1) / kRows;
  if (block < 0 || block >= count) return;
  Work w{};
  const int64_t h0 = int64_t(kvh) * a.group;
  w.query = static_cast<const uint16_t*>(a.query) + first * a.q_tok_stride + h0 * a.q_head_stride;
  w.q_tok_stride = a.q_tok_stride;
  w.q_head_stride = a.q_head_stride;
  w.out = static_cast<uint16_t*>(a.out) + first * a.o_tok_stride + h0 * a.o_head_stride;
  w.o_tok_stride = a.o_tok_stride;
  w.o_head_stride = a.o_head_stride;
  w.group = a.group;
  w.rows = int(len * a.group);
  w.row0 = int(count - 1 - block) * kRows;  // the longest walks first
  w.row0_tok = int(uint32_t(w.row0) / uint32_t(a.group));
  w.base = 0;
  w.t_begin = 0;
  w.t_end = int(uint32_t(min(w.row0 + kRows, w.rows) - 1) / uint32_t(a.group)) + 1;
  w.scale = a.scale;
  w.softcap = a.softcap;
  w.key = static_cast<const uint16_t*>(a.key) + first * a.k_tok_stride + int64_t(kvh) * a.k_head_stride;
  w.value = static_cast<const uint16_t*>(a.value) + first * a.v_tok_stride + int64_t(kvh) * a.v_head_stride;
  w.k_tok_stride = a.k_tok_stride;
  w.v_tok_stride = a.v_tok_stride;
  w.len = int(len);
  attend<kSrcPacked, 0, F16, F16, HD, 1, CAP>(w, lds);
}

template <bool F16, int HD>
hipError_t launch(PackedAttnArgs a, hipStream_t stream) {
  a.blocks = a.num_seqs > 0 ? a.total_tokens * a.group / kRows + a.num_seqs : 0;
  a.tail_blocks = a.zero_tail ? 32 : 0;
  const int64_t grid = (a.blocks + a.tail_blocks) * a.kv_heads;
  if (grid <= 0) return hipSuccess;
  if (grid > 0x7FFFFFFF) return hipErrorInvalidValue;
  if (a.softcap > 0.0f)
    hipLaunchKernelGGL((packed_attention_kernel<F16, HD, true>), dim3(unsigned(grid)), dim3(64 * kWaves), 0, stream, a);
  else
    hipLaunchKernelGGL((packed_attention_kernel<F16, HD, false>), dim3(unsigned(grid)), dim3(64 * kWaves), 0, stream, a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_packed_attention(const PackedAttnArgs& a, int dtype, int64_t head_dim, hipStream_t stream) {
  if (a.total_tokens == 0) return hipSuccess;
  if (dtype == kDtBf16) return head_dim == 128 ? launch<false, 128>(a, stream) : launch<false, 64>(a, stream);
  return head_dim == 128 ? launch<true, 128>(a, stream) : launch<true, 64>(a, stream);
}

}  // namespace llmopt
