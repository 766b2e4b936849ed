/*
 * llmopt_kvq.h -- C ABI of the 8-bit KV cache (quantizing writes, attention over it) and of attention over
 * packed prompts in libllmopt_qlinear.so (gfx950). Same conventions as llmopt_qlinear.h: device pointers owned by the
 * caller, `stream` a hipStream_t as void*, LLMOPT_OK or a negative LLMOPT_ERR_* code, dtype codes
 * LLMOPT_DTYPE_*; the message of a failed call of this header is in llmopt_kvq_last_error() (per host thread).
 *
 * One layer's cache, for keys and for values each:
 *   codes  [num_blocks, kv_heads, block_size, head_dim], one byte each: int8 or e4m3 (OCP, no infinities)
 *   scales [num_blocks, kv_heads] fp32, as written powers of two: a code stands for code x scale. 0: nothing but zeros
 *          was written; NaN: something infinite or NaN was, and the block's numbers of that head read as NaN. Other
 *          positive scales of the caller's are read alike (LLMOPT_KVQ_ALGO_TILES rounds code x scale to bf16).
 * Token t of sequence s lives in block block_ids[s * ldb + t / block_size] at slot t % block_size. block_ids, token
 * offsets, lengths and cu_seqlens are int32. No counterpart in the reference, whose cache holds 16- and 32-bit
 * numbers (src/llmopt/cache/paged_cache.py:137-331); the tables and lengths are its own.
 */
#ifndef LLMOPT_KVQ_H_
#define LLMOPT_KVQ_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define LLMOPT_KVQ_INT8 0
#define LLMOPT_KVQ_E4M3 1

/* The kernel of an attention call: chosen by a rule on the sizes, or one of them. */
#define LLMOPT_KVQ_ALGO_AUTO 0
#define LLMOPT_KVQ_ALGO_ROWS 1  /* 16 query rows per workgroup, keys from memory into registers */
#define LLMOPT_KVQ_ALGO_TILES 2 /* 128 query rows per workgroup, keys in LDS; fp16 and bf16, 16-byte aligned rows */

const char* llmopt_kvq_last_error(void);

/*
 * Quantizes new keys and values into the cache. Element (s, j, h, d) of keys is at s * k_seq_stride + j * k_tok_stride
 * + h * k_head_stride + d, of values likewise, in src_dtype. Uniform rows (cu_seqlens null): sequence s writes its
 * tokens j < min(q_len, query_lens[s]) (query_lens null: q_len) at positions token_offsets[s] + j. Packed rows
 * (cu_seqlens [num_seqs + 1], from 0, not falling): it writes rows cu_seqlens[s] .. cu_seqlens[s + 1] - 1 of
 * [total_tokens, kv_heads, head_dim] (the seq strides are not used, q_len is ignored).
 *
 * Per (block, KV head), with top = 127 (int8) or 448 (e4m3): the new numbers need the scale 2^e, the smallest
 * e >= -126 with max |x| <= top 2^e (0 for all zeros, NaN if one is not finite). A write that holds the block's slot 0
 * starts the block anew with that scale, its other slots unspecified; any other keeps the larger of the old and the
 * needed scale, and where it grew, the block's other slots are rounded to it. A code is x / scale rounded to nearest,
 * ties to even (0 under a NaN scale).
 *
 * A sequence stops at its table row's first negative block or at the end of the row; a block id >= num_blocks and a
 * negative offset write nothing. A block written by two sequences of one call holds unspecified codes afterwards.
 */
int llmopt_kvq_write(void* key_codes, float* key_scales, void* value_codes, float* value_scales, int format,
                     int64_t num_blocks, int64_t block_size, int64_t kv_heads, int64_t head_dim,
                     const int32_t* block_ids, int64_t ldb, const int32_t* token_offsets, const int32_t* cu_seqlens,
                     const int32_t* query_lens, const void* keys, int64_t k_seq_stride, int64_t k_tok_stride,
                     int64_t k_head_stride, const void* values, int64_t v_seq_stride, int64_t v_tok_stride,
                     int64_t v_head_stride, int src_dtype, int64_t num_seqs, int64_t q_len, int64_t total_tokens,
                     void* stream);

/* Bytes of workspace llmopt_kvq_attention uses to split the context (0: no split). */
size_t llmopt_kvq_attention_workspace(int64_t num_seqs, int64_t num_heads, int64_t kv_heads, int64_t head_dim,
                                      int64_t q_len, int64_t ldb, int64_t block_size, int q_dtype, int algo);

/*
 * Attention of q_len query tokens per sequence over the cache, with the rules of llmopt_paged_attention_decode / _prefill
 * (llmopt_attention.h): query token j of sequence s sits at position context_lens[s] - q_len + j and sees the keys
 * t <= that position, t < context_lens[s], whose block id names a block; query head h reads KV head h / (num_heads /
 * kv_heads); zeros without keys; softcap > 0 applies tanh(x / softcap) * softcap to the scaled scores. query
 * element (s, h, j, d) at s * q_seq_stride + h * q_head_stride + j * q_tok_stride + d, out likewise with the o_*
 * strides, in q_dtype (F32, F16 or BF16). Supported: head_dim 64 or 128, any number of heads per KV head, and for
 * LLMOPT_KVQ_ALGO_TILES what it names; otherwise LLMOPT_ERR_UNSUPPORTED. With less workspace than
 * llmopt_kvq_attention_workspace asks for, the context is not split (correct, slower for few sequences).
 */
int llmopt_kvq_attention(const void* query, int q_dtype, int64_t q_seq_stride, int64_t q_head_stride,
                         int64_t q_tok_stride, const void* key_codes, const float* key_scales, const void* value_codes,
                         const float* value_scales, int format, int64_t num_blocks, int64_t block_size,
                         int64_t kv_heads, int64_t head_dim, const int32_t* block_ids, int64_t ldb,
                         const int32_t* context_lens, int64_t num_seqs, int64_t num_heads, int64_t q_len, float scale,
                         float softcap, void* out, int64_t o_seq_stride, int64_t o_head_stride, int64_t o_tok_stride,
                         int algo, void* workspace, size_t workspace_bytes, void* stream);

/*
 * Causal attention over packed prompts: sequence s is rows cu_seqlens[s] .. cu_seqlens[s + 1] - 1 of query
 * [total_tokens, num_heads, head_dim] and key / value [total_tokens, kv_heads, head_dim] (token and head strides in
 * elements, all of dtype F16 or BF16); a token sees its sequence's tokens up to itself. cu_seqlens starts at 0
 * and does not fall. Rows behind the last sequence are cleared in out (zero_tail) or left as they are. out shares no
 * memory with query, key or value, nor one of its rows with another. Supported:
 * head_dim 64 or 128, any number of heads per KV head, every row 16-byte aligned (pointers and strides); otherwise
 * LLMOPT_ERR_UNSUPPORTED.
 */
int llmopt_packed_attention(const void* query, int64_t q_tok_stride, int64_t q_head_stride, const void* key,
                            int64_t k_tok_stride, int64_t k_head_stride, const void* value, int64_t v_tok_stride,
                            int64_t v_head_stride, int dtype, const int32_t* cu_seqlens, int64_t num_seqs,
                            int64_t total_tokens, int64_t num_heads, int64_t kv_heads, int64_t head_dim, float scale,
                            float softcap, void* out, int64_t o_tok_stride, int64_t o_head_stride, int zero_tail,
                            void* stream);

#ifdef __cplusplus
}
#endif

#endif /* LLMOPT_KVQ_H_ */
