// Attention of a chunk of query tokens per sequence over the 8-bit KV cache: the tile kernel of tile_attention.hpp
// over codes that it dequantizes exactly to bf16. fp16 queries: keys as fp16 operands, probabilities in two bf16 pieces. Few row
// blocks (one long prompt's next chunk) are cut along the keys as well, and the parts merged as the decode kernel's are.
//
// Bound by issue: each of a CU's workgroups dequantizes its own tiles (a conversion per two codes, for int8 as many scalings, then
// 16-byte LDS stores), beside the softmax and the MFMAs. Measured (MI355X, 32 query and 8 KV heads of 128, e4m3 codes,
// bf16): the next 512 tokens of 4 prompts of up to 4012 tokens 123 - 134 us (752 - 820 TFLOP/s), by the scaled pair conversion
// of e4m3 codes (163 by way of fp32) and by stepping through the table without a division (4 % of 135). Heads of 64 run three
// workgroups per CU, heads of 128 two. The same chunks, contexts of 2507 - 4012, back to back in a graph (us; with a soft cap of
// 30, of 100):
//   bf16 e4m3, heads of 128 123 (164, 213)    heads of 64 80 (125, 180)
//   bf16 int8              140 (179, 238)                90 (138, 195)
//   fp16 e4m3              169 (200, 254)               113 (159, 217)
//   fp16 int8              184 (218, 270)               122 (170, 223)
#include "tile_attention.hpp"

namespace llmopt {
namespace {

using namespace tile;

template <int FMT, bool QF16, int HD, bool CAP>
__global__ void __launch_bounds__(64 * kWaves) __attribute__((amdgpu_waves_per_eu(HD == 64 ? 3 : 2, HD == 64 ? 3 : 2)))
    kvq_chunk_kernel(const KvqAttnArgs a) {
  __shared__ __align__(16) uint8_t lds[4 * kKeys * HD * 2 + (QF16 ? 2 * kKeys * 4 : 0)];
  // Workgroups in the order (KV head, row block, sequence), a sequence's last blocks (the longest walks) first.
  const uint32_t kv_heads = uint32_t(a.c.kv_heads);
  const int rows = a.group * int(a.q_len);
  const uint32_t blocks = uint32_t((rows + kRows - 1) / kRows);
  const uint32_t rest = blockIdx.x / kv_heads;
  const uint32_t kvh = blockIdx.x - rest * kv_heads;
  const int64_t s = rest / blocks;
  const int row0 = int(blocks - 1 - rest % blocks) * kRows;
  Work w{};
  const int64_t h0 = int64_t(kvh) * a.group;
  w.query = static_cast<const uint16_t*>(a.query) + s * a.q_seq_stride + h0 * a.q_head_stride;
  w.q_tok_stride = a.q_tok_stride;
  w.q_head_stride = a.q_head_stride;
  w.out = static_cast<uint16_t*>(a.out) + s * a.o_seq_stride + h0 * a.o_head_stride;
  w.o_tok_stride = a.o_tok_stride;
  w.o_head_stride = a.o_head_stride;
  w.group = a.group;
  w.rows = rows;
  w.row0 = row0;
  w.row0_tok = int(uint32_t(row0) / uint32_t(a.group));
  w.base = max(a.context_lens[s], 0) - int(a.q_len);
  const int last = int(uint32_t(min(row0 + kRows, rows) - 1) / uint32_t(a.group));
  w.t_end = max(0, min(w.base + last + 1, int(a.c.ldb * a.c.block_size)));
  if (a.splits > 1) {
    const int span = int(a.tiles_per_split) * 32;  // a multiple of 64
    w.t_begin = int(blockIdx.y) * span;
    if (w.t_begin >= w.t_end) return;  // the merge does not read this part
    w.t_end = min(w.t_end, w.t_begin + span);
    const int64_t part = ((int64_t(blockIdx.y) * a.num_seqs + s) * kv_heads + kvh) * rows;
    w.part_out = a.part_out + part * HD;
    w.part_lse = a.part_lse + part;
  }
  w.scale = a.scale;
  w.softcap = a.softcap;
  for (int k = 0; k < 2; ++k) w.codes[k] = a.c.codes[k], w.scales[k] = a.c.scales[k];
  w.table = a.c.block_ids + s * a.c.ldb;
  w.kv_heads = kv_heads;
  w.kvh = kvh;
  w.block_size = uint32_t(a.c.block_size);
  w.ldb = uint32_t(a.c.ldb);
  w.num_blocks = uint32_t(a.c.num_blocks);
  attend<kSrcCodes, FMT, false, QF16, HD, QF16 ? 2 : 1, CAP>(w, lds);
}

template <int FMT, bool QF16, bool CAP>
hipError_t launch_hd(const KvqAttnArgs& a, hipStream_t stream) {
  const int64_t blocks = (a.group * a.q_len + kRows - 1) / kRows;
  const int64_t grid = blocks * a.c.kv_heads * a.num_seqs;
  if (grid > 0x7FFFFFFF) return hipErrorInvalidValue;
  const dim3 grid3(unsigned(grid), unsigned(a.splits));
  if (a.c.head_dim == 128)
    hipLaunchKernelGGL((kvq_chunk_kernel<FMT, QF16, 128, CAP>), grid3, dim3(64 * kWaves), 0, stream, a);
  else
    hipLaunchKernelGGL((kvq_chunk_kernel<FMT, QF16, 64, CAP>), grid3, dim3(64 * kWaves), 0, stream, a);
  if (a.splits > 1) return launch_kvq_merge(a, QF16 ? kDtF16 : kDtBf16, stream);
  return hipGetLastError();
}

template <int FMT>
hipError_t launch_type(const KvqAttnArgs& a, int q_dtype, hipStream_t stream) {
  const bool cap = a.softcap > 0.0f;
  if (q_dtype == kDtF16) return cap ? launch_hd<FMT, true, true>(a, stream) : launch_hd<FMT, true, false>(a, stream);
  return cap ? launch_hd<FMT, false, true>(a, stream) : launch_hd<FMT, false, false>(a, stream);
}

}  // namespace

hipError_t launch_kvq_chunk(const KvqAttnArgs& a, int fmt, int q_dtype, hipStream_t stream) {
  if (a.num_seqs == 0 || a.q_len == 0) return hipSuccess;
  return fmt == kFmtInt8 ? launch_type<kFmtInt8>(a, q_dtype, stream) : launch_type<kFmtE4m3>(a, q_dtype, stream);
}

}  // namespace llmopt
