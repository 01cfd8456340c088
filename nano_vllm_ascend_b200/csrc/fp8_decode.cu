// Paged decode attention over the 8-bit KV pool, one query token a sequence.
// The pool's format is in fp8_kv.cuh.
#include "fp8_attention.cuh"

extern "C" int nvk_fp8_paged_decode_workspace_size(int num_heads, int num_kv_heads, int head_dim, int num_ctas,
                                                   size_t* bytes) {
  *bytes = 4096;
  return NVK_OK;
}

extern "C" int nvk_fp8_paged_decode(void* out, const void* query, const void* kv_cache, int num_blocks,
                                    int block_size, const int32_t* block_tables, int block_table_stride,
                                    int max_blocks_per_seq, const int32_t* context_lens, int batch, int num_heads,
                                    int num_kv_heads, int head_dim, float scale, int num_ctas, void* workspace,
                                    size_t workspace_bytes, int* error_word, nvk_stream_t stream) {
  using namespace nvk;
  const char* who = "fp8_paged_decode";
  if (batch < 0 || num_heads <= 0) return fail(NVK_ERR_INVALID_ARGUMENT, "%s: batch %d", who, batch);
  int rc = fp8::check_pool(kv_cache, num_blocks, block_size, num_kv_heads, head_dim, who);
  if (rc != NVK_OK) return rc;
  if (!(scale > 0.f)) return fail(NVK_ERR_INVALID_ARGUMENT, "%s: scale %g is not positive", who, double(scale));
  if (max_blocks_per_seq <= 0 || block_table_stride < max_blocks_per_seq)
    return fail(NVK_ERR_INVALID_ARGUMENT, "%s: block table stride %d below its %d columns", who, block_table_stride,
                max_blocks_per_seq);
  if (batch == 0) return NVK_OK;
  if (!out || !query || !block_tables || !context_lens || !workspace)
    return fail(NVK_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
  fp8::AttentionArgs a{static_cast<__nv_bfloat16*>(out), static_cast<const __nv_bfloat16*>(query),
                       static_cast<const uint8_t*>(kv_cache), block_tables, context_lens, nullptr,
                       error_word ? error_word : static_cast<int*>(workspace), batch, batch, num_heads, num_kv_heads,
                       block_table_stride, max_blocks_per_seq, num_blocks, fp8::units_log2(block_size),
                       scale * 1.4426950408889634f};
  return fp8::launch_attention(a, reinterpret_cast<cudaStream_t>(stream), "fp8_paged_decode launch");
}
