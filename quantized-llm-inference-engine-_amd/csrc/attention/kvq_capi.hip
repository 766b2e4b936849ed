// C ABI of llmopt_kvq.h: checks, work split and launches of the 8-bit KV cache and of packed prompts.
#include <stdarg.h>
#include <stdio.h>

#include <algorithm>

#include "../../../include/llmopt_kvq.h"
#include "../../../include/llmopt_qlinear.h"
#include "attn_common.hpp"

namespace {

thread_local char g_error[512];

int fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
int fail(int code, const char* fmt, ...) {
  va_list args;
  va_start(args, fmt);
  vsnprintf(g_error, sizeof(g_error), fmt, args);
  va_end(args);
  return code;
}

int hip_status(hipError_t err, const char* what) {
  if (err == hipSuccess) return LLMOPT_OK;
  return fail(LLMOPT_ERR_HIP, "%s: %s", what, hipGetErrorString(err));
}

bool valid_dtype(int dt) { return dt == LLMOPT_DTYPE_F32 || dt == LLMOPT_DTYPE_F16 || dt == LLMOPT_DTYPE_BF16; }

bool aligned(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

constexpr int64_t kMaxInt = 0x7FFFFFFF;

int describe_cache(llmopt::KvqCache& c, const void* key_codes, const float* key_scales, const void* value_codes,
                   const float* value_scales, int format, int64_t num_blocks, int64_t block_size, int64_t kv_heads,
                   int64_t head_dim, const int32_t* block_ids, int64_t ldb) {
  if (format != LLMOPT_KVQ_INT8 && format != LLMOPT_KVQ_E4M3)
    return fail(LLMOPT_ERR_INVALID_ARG, "bad cache format code %d", format);
  if (num_blocks < 1 || block_size < 1 || kv_heads < 1 || head_dim < 1 || ldb < 0)
    return fail(LLMOPT_ERR_INVALID_ARG,
                "bad cache geometry: blocks %lld, block_size %lld, kv_heads %lld, head_dim %lld, table width %lld",
                (long long)num_blocks, (long long)block_size, (long long)kv_heads, (long long)head_dim, (long long)ldb);
  // Rows of head_dim codes have 32-bit numbers (their bytes 64-bit offsets), and so do a table row's tokens.
  if (kv_heads > 65535 || block_size > kMaxInt / 4 || head_dim > 65536 || block_size * head_dim > kMaxInt / 4 ||
      num_blocks > kMaxInt / (kv_heads * block_size))
    return fail(LLMOPT_ERR_UNSUPPORTED, "cache of %lld blocks x %lld heads x %lld tokens too large for 32-bit row numbers",
                (long long)num_blocks, (long long)kv_heads, (long long)block_size);
  if (ldb > 0 && ldb >= kMaxInt / 2 / block_size)
    return fail(LLMOPT_ERR_UNSUPPORTED, "block table row of %lld blocks too long", (long long)ldb);
  c.codes[0] = static_cast<uint8_t*>(const_cast<void*>(key_codes));
  c.codes[1] = static_cast<uint8_t*>(const_cast<void*>(value_codes));
  c.scales[0] = const_cast<float*>(key_scales);
  c.scales[1] = const_cast<float*>(value_scales);
  c.num_blocks = num_blocks;
  c.block_size = block_size;
  c.kv_heads = kv_heads;
  c.head_dim = head_dim;
  c.block_ids = block_ids;
  c.ldb = ldb;
  return LLMOPT_OK;
}

// How the attention's work is cut: on the tile kernel or the decode kernel (`waves` per workgroup), in `splits` of the
// context of `tiles_per_split` 32-token tiles each. The context lengths are on the device, so the table's width stands for
// them. Measured (MI355X, bf16, 32 / 8 heads of 128, int8, ragged contexts of half to the whole width; us):
//   * Tile or decode kernel: the decode kernel reads the keys once per 16 query rows, the tile kernel once per 128, but it
//     starts slower and its workgroups are fewer. Level where (16-row blocks x 32-token tiles) is about 28000 at heads of
//     128 (half the work each at 64): 1 sequence of 8000, 32 / 64 / 512 new tokens 26.6 / 39.6 / 219 against 30.9 / 33.3 /
//     112; 8 of 2000, 24 / 64 tokens 34.2 / 55 against 32.9 / 46; 32 of 1000, 9 / 24 tokens 34.4 / 51 against 34.7 / 43.
//   * Workgroups of eight waves, one per CU, in one round: 1 sequence of 8000 in 32 splits 14.2 (4 splits 23.5), 8 of 4096
//     in 4 splits 19.6 (1 33, 8 23.3), 32 of 640 in 1 split 12.5 (2 19.2); past 256 pairs none (64 of 8192: 147 - 165; 2
//     splits 176). A split has a tile per wave at least, and up to 24 tiles stay whole but for a few pairs: the merge costs 3.
//   * Short contexts, the rule's splits against one, in a graph: 1 sequence of 384 (2 splits) 8.2 against 7.1, of 512 (2) 8.4 against
//     8.0, of 641 (3) 8.5 against 9.9, of 1024 (4) 8.5 against 11.8; 2 and 3 sequences alike; 8 of 800 (4) 9.0 against 10.7, of 1024
//     9.2 against 12.1; 16 of 800 (2) 11.6 against 10.9, of 1024 12.2 against 13.3. Up to 256 tokens there is one. Where a pair has 12 - 16
//     tiles, or 16 sequences 25, one split would be 0.4 - 1.1 faster.
//   * Four waves, two workgroups per CU, from 512 pairs over tables of up to 2048 tokens: 64 of 640 18.0 (eight waves 21.4),
//     128 of 1024 47 (57), 64 of 2048 45.7 (46.3); longer ones 162 (147).
//   * Tables much wider than their contexts: a split is at most 1024 tokens for a few pairs, 8192 for many.
//   * The tile kernel's row blocks fill two workgroups per CU with splits of 512 tokens at least: 1 sequence of 8000, 512
//     tokens 224 without splits, 112 with.
struct Plan {
  bool tile;
  int splits, waves;
  int64_t tiles_per_split;
};

Plan plan_attention(int64_t num_seqs, int64_t kv_heads, int64_t group, int64_t head_dim, int64_t q_len, int64_t ldb,
                    int64_t block_size, int q_dtype, bool tile_rows, int algo) {
  const int64_t tiles = std::max<int64_t>(1, (ldb * block_size + 31) / 32), rows = group * q_len;
  const int64_t pairs = std::max<int64_t>(1, num_seqs * kv_heads * ((rows + 15) / 16));
  const bool tile = algo == LLMOPT_KVQ_ALGO_TILES ||
                    (algo == LLMOPT_KVQ_ALGO_AUTO && tile_rows && q_dtype != LLMOPT_DTYPE_F32 && rows > 32 &&
                     pairs * tiles * head_dim > 3600000);
  if (tile) {
    const int64_t blocks = num_seqs * kv_heads * ((rows + 127) / 128);
    int64_t splits = std::max<int64_t>(1, std::min<int64_t>({512 / blocks, tiles / 16, 16}));
    const int64_t per = ((tiles + splits - 1) / splits + 1) / 2 * 2;
    return Plan{true, int((tiles + per - 1) / per), 4, per};
  }
  const int waves = pairs >= 512 && tiles <= 64 ? 4 : 8;
  int64_t splits = 1;
  if (pairs < 256 && (tiles > 24 || pairs < 32)) splits = std::max<int64_t>(1, std::min(256 / pairs, (tiles + 7) / 8));
  splits = std::max(splits, tiles / (pairs <= 32 ? 32 : pairs < 256 ? 128 : 256));
  splits = std::min<int64_t>(splits, 256);
  const int64_t per = (tiles + splits - 1) / splits;
  return Plan{false, int((tiles + per - 1) / per), waves, per};
}

// A workgroup of the tile kernel reads its query rows (128 tokens, one KV head's query heads) and writes its output at
// 32-bit offsets, and finds a row's token in fp32.
bool near_rows(int64_t group, int64_t tok_stride, int64_t head_stride) {
  return group < (int64_t(1) << 19) && tok_stride >= 0 && tok_stride <= (int64_t(1) << 22) && head_stride >= 0 && head_stride <= (int64_t(1) << 29) / group;
}

}  // namespace

extern "C" {

const char* llmopt_kvq_last_error(void) { return g_error; }

int llmopt_kvq_write(void* key_codes, float* key_scales, void* value_codes, float* value_scales, int format,
                     int64_t num_blocks, int64_t block_size, int64_t kv_heads, int64_t head_dim,
                     const int32_t* block_ids, int64_t ldb, const int32_t* token_offsets, const int32_t* cu_seqlens,
                     const int32_t* query_lens, const void* keys, int64_t k_seq_stride, int64_t k_tok_stride,
                     int64_t k_head_stride, const void* values, int64_t v_seq_stride, int64_t v_tok_stride,
                     int64_t v_head_stride, int src_dtype, int64_t num_seqs, int64_t q_len, int64_t total_tokens,
                     void* stream) {
  llmopt::KvqWriteArgs a{};
  const int rc = describe_cache(a.c, key_codes, key_scales, value_codes, value_scales, format, num_blocks, block_size,
                                kv_heads, head_dim, block_ids, ldb);
  if (rc != LLMOPT_OK) return rc;
  if (!valid_dtype(src_dtype)) return fail(LLMOPT_ERR_INVALID_ARG, "bad dtype code %d", src_dtype);
  if (num_seqs < 0 || q_len < 0 || total_tokens < 0)
    return fail(LLMOPT_ERR_INVALID_ARG, "negative sequence count, q_len or token count");
  const bool packed = cu_seqlens != nullptr;
  if (num_seqs == 0 || ldb == 0 || (packed ? total_tokens : q_len) == 0) return LLMOPT_OK;
  if (!key_codes || !value_codes || !key_scales || !value_scales || !block_ids || !token_offsets || !keys || !values)
    return fail(LLMOPT_ERR_INVALID_ARG, "null pointer argument");
  if (num_seqs > kMaxInt / 4 || q_len > kMaxInt / 2 || total_tokens > kMaxInt / 2)
    return fail(LLMOPT_ERR_UNSUPPORTED, "too many sequences or tokens for one launch");
  a.offsets = token_offsets;
  a.cu_seqlens = cu_seqlens;
  a.query_lens = query_lens;
  a.src[0] = keys;
  a.src[1] = values;
  a.seq_stride[0] = k_seq_stride, a.tok_stride[0] = k_tok_stride, a.head_stride[0] = k_head_stride;
  a.seq_stride[1] = v_seq_stride, a.tok_stride[1] = v_tok_stride, a.head_stride[1] = v_head_stride;
  a.num_seqs = num_seqs;
  a.q_len = q_len;
  a.total_tokens = total_tokens;
  a.units_per_seq = (q_len + block_size - 2) / block_size + 1;  // blocks that q_len tokens can touch
  a.units = packed ? total_tokens / block_size + 2 * num_seqs : num_seqs * a.units_per_seq;
  if (a.units * ((2 * kv_heads + 3) / 4) > kMaxInt)
    return fail(LLMOPT_ERR_UNSUPPORTED, "too many sequences or tokens for one launch");
  const int64_t esize = src_dtype == LLMOPT_DTYPE_F32 ? 4 : 2;
  bool vec = head_dim % 8 == 0 && aligned(key_codes, 8) && aligned(value_codes, 8);
  for (int k = 0; k < 2; ++k)
    vec = vec && aligned(a.src[k], 16) && (a.tok_stride[k] * esize) % 16 == 0 && (a.head_stride[k] * esize) % 16 == 0 &&
          (packed || (a.seq_stride[k] * esize) % 16 == 0);
  return hip_status(llmopt::launch_kvq_write(a, format, src_dtype, vec, static_cast<hipStream_t>(stream)),
                    "quantizing kv write launch");
}

size_t llmopt_kvq_attention_workspace(int64_t num_seqs, int64_t num_heads, int64_t kv_heads, int64_t head_dim,
                                      int64_t q_len, int64_t ldb, int64_t block_size, int q_dtype, int algo) {
  if (num_seqs <= 0 || num_heads <= 0 || kv_heads <= 0 || head_dim <= 0 || q_len <= 0 || ldb <= 0 || block_size <= 0)
    return 0;
  if (num_heads % kv_heads != 0) return 0;
  const Plan plan = plan_attention(num_seqs, kv_heads, num_heads / kv_heads, head_dim, q_len, ldb, block_size, q_dtype, true, algo);
  if (plan.splits <= 1) return 0;
  return size_t(plan.splits) * size_t(num_seqs) * size_t(num_heads) * size_t(q_len) * size_t(head_dim + 1) * sizeof(float);
}

int llmopt_kvq_attention(const void* query, int q_dtype, int64_t q_seq_stride, int64_t q_head_stride,
                         int64_t q_tok_stride, const void* key_codes, const float* key_scales, const void* value_codes,
                         const float* value_scales, int format, int64_t num_blocks, int64_t block_size,
                         int64_t kv_heads, int64_t head_dim, const int32_t* block_ids, int64_t ldb,
                         const int32_t* context_lens, int64_t num_seqs, int64_t num_heads, int64_t q_len, float scale,
                         float softcap, void* out, int64_t o_seq_stride, int64_t o_head_stride, int64_t o_tok_stride,
                         int algo, void* workspace, size_t workspace_bytes, void* stream) {
  llmopt::KvqAttnArgs a{};
  const int rc = describe_cache(a.c, key_codes, key_scales, value_codes, value_scales, format, num_blocks, block_size,
                                kv_heads, head_dim, block_ids, ldb);
  if (rc != LLMOPT_OK) return rc;
  if (!valid_dtype(q_dtype)) return fail(LLMOPT_ERR_INVALID_ARG, "bad dtype code %d", q_dtype);
  if (algo < LLMOPT_KVQ_ALGO_AUTO || algo > LLMOPT_KVQ_ALGO_TILES)
    return fail(LLMOPT_ERR_INVALID_ARG, "bad algorithm code %d", algo);
  if (num_seqs < 0 || q_len < 0 || num_heads < 1 || num_heads % kv_heads != 0)
    return fail(LLMOPT_ERR_INVALID_ARG, "num_heads %lld must be a positive multiple of kv_heads %lld, sequences and "
                "q_len not negative", (long long)num_heads, (long long)kv_heads);
  if (head_dim != 64 && head_dim != 128)
    return fail(LLMOPT_ERR_UNSUPPORTED, "attention over the 8-bit cache: head_dim %lld", (long long)head_dim);
  if (num_seqs == 0 || q_len == 0) return LLMOPT_OK;
  if (!query || !key_codes || !value_codes || !key_scales || !value_scales || (!block_ids && ldb > 0) || !context_lens ||
      !out)
    return fail(LLMOPT_ERR_INVALID_ARG, "null pointer argument");
  const int64_t group = num_heads / kv_heads;
  if (num_seqs > 65535 || q_len > kMaxInt / 4 || group * q_len > kMaxInt / 4)
    return fail(LLMOPT_ERR_UNSUPPORTED, "batch of %lld sequences x %lld tokens too large for one launch",
                (long long)num_seqs, (long long)q_len);
  if (!aligned(key_codes, 16) || !aligned(value_codes, 16))
    return fail(LLMOPT_ERR_UNSUPPORTED, "caches must be 16-byte aligned");
  a.query = query;
  a.q_seq_stride = q_seq_stride, a.q_head_stride = q_head_stride, a.q_tok_stride = q_tok_stride;
  a.out = out;
  a.o_seq_stride = o_seq_stride, a.o_head_stride = o_head_stride, a.o_tok_stride = o_tok_stride;
  a.context_lens = context_lens;
  a.num_seqs = num_seqs;
  a.num_heads = num_heads;
  a.q_len = q_len;
  a.group = int(group);
  a.scale = scale;
  a.softcap = softcap;
  const int64_t esize = q_dtype == LLMOPT_DTYPE_F32 ? 4 : 2;
  auto rows16 = [&](const void* p, int64_t x, int64_t y, int64_t z) {
    return aligned(p, 16) && (x * esize) % 16 == 0 && (y * esize) % 16 == 0 && (z * esize) % 16 == 0;
  };
  a.q_vec = rows16(query, q_seq_stride, q_head_stride, q_tok_stride);
  const bool tile_rows = a.q_vec && near_rows(group, q_tok_stride, q_head_stride) &&
                         near_rows(group, o_tok_stride, o_head_stride) && rows16(out, o_seq_stride, o_head_stride, o_tok_stride);
  if (algo == LLMOPT_KVQ_ALGO_TILES && (q_dtype == LLMOPT_DTYPE_F32 || !tile_rows))
    return fail(LLMOPT_ERR_UNSUPPORTED, "the tile kernel takes fp16 and bf16 rows aligned to 16 bytes");
  const Plan plan = plan_attention(num_seqs, kv_heads, group, head_dim, q_len, ldb, block_size, q_dtype, tile_rows, algo);
  const int64_t blocks = kv_heads * ((group * q_len + (plan.tile ? 127 : 15)) / (plan.tile ? 128 : 16));
  if (plan.tile ? blocks > kMaxInt / num_seqs : blocks > 65535)
    return fail(LLMOPT_ERR_UNSUPPORTED, "batch of %lld sequences x %lld tokens too large for one launch",
                (long long)num_seqs, (long long)q_len);
  a.waves = plan.waves;
  a.splits = plan.splits;
  a.tiles_per_split = plan.tiles_per_split;
  const size_t rows = size_t(plan.splits) * size_t(num_seqs) * size_t(num_heads) * size_t(q_len);
  if (a.splits > 1 && (workspace == nullptr || workspace_bytes < rows * size_t(head_dim + 1) * sizeof(float) ||
                       !aligned(workspace, 16))) {
    a.splits = 1;
    a.tiles_per_split = std::max<int64_t>(1, (ldb * block_size + 31) / 32);
  }
  if (a.splits > 1) {
    a.part_out = static_cast<float*>(workspace);
    a.part_lse = a.part_out + rows * size_t(head_dim);
  }
  if (plan.tile)
    return hip_status(llmopt::launch_kvq_chunk(a, format, q_dtype, static_cast<hipStream_t>(stream)),
                      "chunk attention launch");
  return hip_status(llmopt::launch_kvq_decode(a, format, q_dtype, static_cast<hipStream_t>(stream)),
                    "attention launch");
}

int llmopt_packed_attention(const void* query, int64_t q_tok_stride, int64_t q_head_stride, const void* key,
                            int64_t k_tok_stride, int64_t k_head_stride, const void* value, int64_t v_tok_stride,
                            int64_t v_head_stride, int dtype, const int32_t* cu_seqlens, int64_t num_seqs,
                            int64_t total_tokens, int64_t num_heads, int64_t kv_heads, int64_t head_dim, float scale,
                            float softcap, void* out, int64_t o_tok_stride, int64_t o_head_stride, int zero_tail,
                            void* stream) {
  if (!valid_dtype(dtype)) return fail(LLMOPT_ERR_INVALID_ARG, "bad dtype code %d", dtype);
  if (num_seqs < 0 || total_tokens < 0 || num_heads < 1 || kv_heads < 1 || num_heads % kv_heads != 0)
    return fail(LLMOPT_ERR_INVALID_ARG, "num_heads %lld must be a positive multiple of kv_heads %lld, sequences and "
                "tokens not negative", (long long)num_heads, (long long)kv_heads);
  if (dtype == LLMOPT_DTYPE_F32 || (head_dim != 64 && head_dim != 128))
    return fail(LLMOPT_ERR_UNSUPPORTED, "packed attention: dtype code %d, head_dim %lld", dtype, (long long)head_dim);
  if (total_tokens == 0) return LLMOPT_OK;
  if (!query || !key || !value || !out || (num_seqs > 0 && !cu_seqlens))
    return fail(LLMOPT_ERR_INVALID_ARG, "null pointer argument");
  const int64_t group = num_heads / kv_heads;
  constexpr int64_t kStride = int64_t(1) << 24;  // a tile's 64 rows at 32-bit offsets
  if (total_tokens > kMaxInt / 4 / group || num_seqs > kMaxInt / 4 || k_tok_stride < 0 || k_tok_stride > kStride ||
      v_tok_stride < 0 || v_tok_stride > kStride ||
      !near_rows(group, q_tok_stride, q_head_stride) || !near_rows(group, o_tok_stride, o_head_stride) ||
      ((total_tokens * group + 127) / 128 + num_seqs + 64) > kMaxInt / kv_heads)
    return fail(LLMOPT_ERR_UNSUPPORTED, "packed attention: %lld tokens, %lld sequences, token strides %lld / %lld / %lld",
                (long long)total_tokens, (long long)num_seqs, (long long)q_tok_stride, (long long)k_tok_stride,
                (long long)v_tok_stride);
  const int64_t strides[] = {q_tok_stride, q_head_stride, k_tok_stride, k_head_stride, v_tok_stride,
                             v_head_stride, o_tok_stride, o_head_stride};
  bool rows16 = aligned(query, 16) && aligned(key, 16) && aligned(value, 16) && aligned(out, 16);
  for (const int64_t s : strides) rows16 = rows16 && s % 8 == 0;
  if (!rows16) return fail(LLMOPT_ERR_UNSUPPORTED, "packed attention: rows must be 16-byte aligned");
  llmopt::PackedAttnArgs a{};
  a.query = query, a.key = key, a.value = value, a.out = out;
  a.q_tok_stride = q_tok_stride, a.q_head_stride = q_head_stride;
  a.k_tok_stride = k_tok_stride, a.k_head_stride = k_head_stride;
  a.v_tok_stride = v_tok_stride, a.v_head_stride = v_head_stride;
  a.o_tok_stride = o_tok_stride, a.o_head_stride = o_head_stride;
  a.cu_seqlens = cu_seqlens;
  a.num_seqs = num_seqs;
  a.total_tokens = total_tokens;
  a.num_heads = num_heads;
  a.kv_heads = kv_heads;
  a.group = int(group);
  a.scale = scale;
  a.softcap = softcap;
  a.zero_tail = zero_tail;
  return hip_status(llmopt::launch_packed_attention(a, dtype, head_dim, static_cast<hipStream_t>(stream)),
                    "packed attention launch");
}

}  // extern "C"
