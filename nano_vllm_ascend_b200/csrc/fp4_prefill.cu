// Causal prefill attention over the 4-bit KV pool (cached prefix and the rows
// appended this step). The kernel body, with its design, is in
// prefill_core.cuh; the pool's format is in fp4_kv.cuh.
//
// Tensor-bound by its operations (4 * 128 a visible pair and head); 82.4 us
// for 32 requests of 256 tokens over 768 cached ones (16 heads on 8, blocks of
// 128; 60.2 GFLOP, 730 TF/s), where the bf16 kernel over 3.6 times the bytes
// takes 71.5: the decoders' instructions and the fetch of the longer code are
// the difference.
#include "prefill_core.cuh"

namespace nvk {
using namespace prefill;
namespace {

__global__ void __launch_bounds__(kThreadsFp4, 1) fp4_prefill_kernel(const __grid_constant__ CUtensorMap qmap,
                                                                     const PrefillArgs a) {
  prefill_body<true>(qmap, qmap, qmap, a);
}

}  // namespace
}  // namespace nvk

extern "C" int nvk_fp4_paged_prefill(void* out, const void* query, const void* kv_cache, int num_blocks,
                                     int block_size, const int32_t* block_tables, int block_table_stride,
                                     int max_blocks_per_seq, const int32_t* cu_seqlens_q, const int32_t* kv_lens,
                                     int batch, int total_q, int max_q_len, int num_heads, int num_kv_heads,
                                     int head_dim, float scale, float k_scale, float v_scale, int* error_word,
                                     nvk_stream_t stream) {
  using namespace nvk;
  const char* who = "fp4_paged_prefill";
  if (batch < 0 || total_q < 0 || max_q_len < 0 || num_heads <= 0)
    return fail(NVK_ERR_INVALID_ARGUMENT, "%s: bad sizes (batch=%d total_q=%d max_q_len=%d heads=%d)", who, batch,
                total_q, max_q_len, num_heads);
  int rc = fp4::check_pool(kv_cache, num_blocks, block_size, num_kv_heads, head_dim, k_scale, v_scale, who);
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
  CUtensorMap qm;
  if ((rc = kv_tensor_map(&qm, query, total_q, num_heads, kRows)) != NVK_OK) return rc;
  PrefillArgs a{};
  a.out = static_cast<__nv_bfloat16*>(out);
  a.block_tables = block_tables;
  a.cu_q = cu_seqlens_q;
  a.kv_lens = kv_lens;
  a.err = error_word;
  a.bt_stride = block_table_stride;
  a.num_blocks = num_blocks;
  a.num_heads = num_heads;
  a.qpk = num_heads / num_kv_heads;
  a.paired = (a.qpk % 2 == 0) ? 1 : 0;
  a.paged = 1;
  a.batch = batch;
  a.qtiles = (max_q_len + kRows - 1) / kRows;
  a.scale_log2 = scale * 1.4426950408889634f * k_scale;
  a.pool = static_cast<const uint8_t*>(kv_cache);
  a.kvh = num_kv_heads;
  a.upb_log2 = fp4::units_log2(block_size);
  a.max_blocks = max_blocks_per_seq;
  a.total_q = total_q;
  a.out_scale = v_scale;
  const size_t smem = sizeof(PrefillSmem) + 1024;
  if ((rc = ensure_dynamic_smem(reinterpret_cast<const void*>(&fp4_prefill_kernel), smem)) != NVK_OK) return rc;
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  const int64_t items = static_cast<int64_t>(a.qtiles) * (num_heads / (a.paired ? kStreams : 1)) * batch;
  if (items > (int64_t(1) << 30))
    return fail(NVK_ERR_UNSUPPORTED, "%s: %lld work items above the kernel's range", who, (long long)items);
  const int grid = static_cast<int>(items < sms ? items : sms);
  return check_cuda(launch_pdl(fp4_prefill_kernel, dim3(grid), dim3(kThreadsFp4), smem,
                               reinterpret_cast<cudaStream_t>(stream), qm, a),
                    "fp4_paged_prefill launch");
}
