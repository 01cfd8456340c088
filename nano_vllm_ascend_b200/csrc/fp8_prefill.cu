// Causal prefill attention over the 8-bit KV pool (cached prefix and the rows
// appended this step). The pool's format is in fp8_kv.cuh.
#include "fp8_attention.cuh"

extern "C" int nvk_fp8_paged_prefill(void* out, const void* query, const void* kv_cache, int num_blocks,
                                     int block_size, const int32_t* block_tables, int block_table_stride,
                                     int max_blocks_per_seq, const int32_t* cu_seqlens_q, const int32_t* kv_lens,
                                     int batch, int total_q, int max_q_len, int num_heads, int num_kv_heads,
                                     int head_dim, float scale, int* error_word, nvk_stream_t stream) {
  using namespace nvk;
  const char* who = "fp8_paged_prefill";
  if (batch < 0 || total_q < 0 || max_q_len < 0 || num_heads <= 0)
    return fail(NVK_ERR_INVALID_ARGUMENT, "%s: bad sizes (batch=%d total_q=%d max_q_len=%d heads=%d)", who, batch,
                total_q, max_q_len, num_heads);
  int rc = fp8::check_pool(kv_cache, num_blocks, block_size, num_kv_heads, head_dim, who);
  if (rc != NVK_OK) return rc;
  if (num_heads % num_kv_heads != 0)
    return fail(NVK_ERR_INVALID_ARGUMENT, "%s: num_heads %d not a multiple of num_kv_heads %d", who, num_heads,
                num_kv_heads);
  if (batch > 65535 || num_heads > 65535)
    return fail(NVK_ERR_UNSUPPORTED, "%s: batch %d or heads %d above grid limit", who, batch, num_heads);
  if (!(scale > 0.f)) return fail(NVK_ERR_INVALID_ARGUMENT, "%s: scale %g is not positive", who, double(scale));
  if (max_blocks_per_seq <= 0 || block_table_stride < max_blocks_per_seq)
    return fail(NVK_ERR_INVALID_ARGUMENT, "%s: block table stride %d below its %d columns", who, block_table_stride,
                max_blocks_per_seq);
  if (batch == 0 || total_q == 0 || max_q_len == 0) return NVK_OK;
  if (!out || !query || !block_tables || !cu_seqlens_q || !kv_lens)
    return fail(NVK_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
  if (!aligned16(out) || !aligned16(query))
    return fail(NVK_ERR_INVALID_ARGUMENT, "%s: q/out must be 16-byte aligned", who);
  fp8::AttentionArgs a{static_cast<__nv_bfloat16*>(out), static_cast<const __nv_bfloat16*>(query),
                       static_cast<const uint8_t*>(kv_cache), block_tables, kv_lens, cu_seqlens_q, error_word, total_q,
                       batch, num_heads, num_kv_heads, block_table_stride, max_blocks_per_seq, num_blocks,
                       fp8::units_log2(block_size), scale * 1.4426950408889634f};
  return fp8::launch_attention(a, reinterpret_cast<cudaStream_t>(stream), "fp8_paged_prefill launch");
}
