// Causal prefill attention over bf16 K and V: the paged pool or contiguous
// rows. The kernel body, with its design, is in prefill_core.cuh.
//
// Replaces torch_npu.npu_fused_infer_attention_score as called from
// src/nanovllm_ascend/layers/npu_prefill_attention.py:82-112 (TND layout,
// sparse_mode=3): paged mode reads the whole KV of a sequence (cached prefix
// + rows appended this step) through its block table with absolute kv
// lengths; dense mode reads contiguous K/V rows delimited by cumulative
// lengths.
#include "prefill_core.cuh"

namespace nvk {
using namespace prefill;
namespace {

__global__ void __maxnreg__(168) prefill_kernel(const __grid_constant__ CUtensorMap qmap,
                                                const __grid_constant__ CUtensorMap kmap,
                                                const __grid_constant__ CUtensorMap vmap, const PrefillArgs a) {
  prefill_body<false>(qmap, kmap, vmap, a);
}

int launch_prefill(const CUtensorMap& qm, const CUtensorMap& km, const CUtensorMap& vm, PrefillArgs a,
                   int max_q_len, cudaStream_t stream) {
  const size_t smem = sizeof(PrefillSmem) + 1024;
  int rc = ensure_dynamic_smem(reinterpret_cast<const void*>(&prefill_kernel), smem);
  if (rc != NVK_OK) return rc;
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  a.qtiles = (max_q_len + kRows - 1) / kRows;
  a.paired = (a.qpk % 2 == 0) ? 1 : 0;
  const int64_t items = static_cast<int64_t>(a.qtiles) * (a.num_heads / (a.paired ? kStreams : 1)) * a.batch;
  if (items > (int64_t(1) << 30))
    return fail(NVK_ERR_UNSUPPORTED, "prefill: %lld work items above the kernel's range", (long long)items);
  const int grid = static_cast<int>(items < sms ? items : sms);
  return check_cuda(launch_pdl(prefill_kernel, dim3(grid), dim3(kThreads), smem, stream, qm, km, vm, a),
                    "prefill launch");
}

int check_common(const void* out, const void* query, int batch, int total_q, int max_q_len, int num_heads,
                 int num_kv_heads, int head_dim, const char* who) {
  if (batch < 0 || total_q < 0 || max_q_len < 0 || num_heads <= 0 || num_kv_heads <= 0)
    return fail(NVK_ERR_INVALID_ARGUMENT, "%s: bad sizes (batch=%d total_q=%d max_q_len=%d heads=%d kv_heads=%d)",
                who, batch, total_q, max_q_len, num_heads, num_kv_heads);
  if (head_dim != kD) return fail(NVK_ERR_UNSUPPORTED, "%s: head_dim %d unsupported (128 only)", who, head_dim);
  if (num_heads % num_kv_heads != 0)
    return fail(NVK_ERR_INVALID_ARGUMENT, "%s: num_heads %d not a multiple of num_kv_heads %d", who, num_heads,
                num_kv_heads);
  if (batch > 65535 || num_heads > 65535)
    return fail(NVK_ERR_UNSUPPORTED, "%s: batch %d or heads %d above grid limit", who, batch, num_heads);
  if (!out || !query) return fail(NVK_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
  if (!aligned16(out) || !aligned16(query))
    return fail(NVK_ERR_INVALID_ARGUMENT, "%s: q/out must be 16-byte aligned", who);
  return NVK_OK;
}

}  // namespace
}  // namespace nvk

extern "C" int nvk_paged_prefill(void* out, const void* query, const void* key_cache, const void* value_cache,
                                 int num_blocks, int block_size, const int32_t* block_tables, int block_table_stride,
                                 const int32_t* cu_seqlens_q, const int32_t* kv_lens, int batch, int total_q,
                                 int max_q_len, int num_heads, int num_kv_heads, int head_dim, float scale,
                                 int* error_word, nvk_stream_t stream) {
  using namespace nvk;
  int rc = check_common(out, query, batch, total_q, max_q_len, num_heads, num_kv_heads, head_dim, "paged_prefill");
  if (rc != NVK_OK) return rc;
  if (batch == 0 || total_q == 0 || max_q_len == 0) return NVK_OK;
  if (block_size != kRows)
    return fail(NVK_ERR_UNSUPPORTED, "paged_prefill: block_size %d unsupported (128 only)", block_size);
  if (num_blocks <= 0 || !key_cache || !value_cache || !block_tables || !cu_seqlens_q || !kv_lens)
    return fail(NVK_ERR_INVALID_ARGUMENT, "paged_prefill: null pointer or empty pool");
  if (block_table_stride <= 0) return fail(NVK_ERR_INVALID_ARGUMENT, "paged_prefill: bad block table stride");
  CUtensorMap qm, km, vm;
  if ((rc = kv_tensor_map(&qm, query, total_q, num_heads, kRows)) != NVK_OK) return rc;
  const int64_t rows = static_cast<int64_t>(num_blocks) * block_size;
  if ((rc = kv_tensor_map(&km, key_cache, rows, num_kv_heads, kKeys)) != NVK_OK) return rc;
  if ((rc = kv_tensor_map(&vm, value_cache, rows, num_kv_heads, kKeys)) != NVK_OK) return rc;
  PrefillArgs a{};
  a.out = static_cast<__nv_bfloat16*>(out);
  a.block_tables = block_tables;
  a.cu_q = cu_seqlens_q;
  a.kv_lens = kv_lens;
  a.cu_kv = nullptr;
  a.err = error_word;
  a.bt_stride = block_table_stride;
  a.num_blocks = num_blocks;
  a.num_heads = num_heads;
  a.qpk = num_heads / num_kv_heads;
  a.paged = 1;
  a.batch = batch;
  a.scale_log2 = scale * 1.4426950408889634f;
  return launch_prefill(qm, km, vm, a, max_q_len, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int nvk_dense_prefill(void* out, const void* query, const void* key, const void* value,
                                 const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_kv, int batch, int total_q,
                                 int total_kv, int max_q_len, int num_heads, int num_kv_heads, int head_dim,
                                 float scale, int* error_word, nvk_stream_t stream) {
  using namespace nvk;
  int rc = check_common(out, query, batch, total_q, max_q_len, num_heads, num_kv_heads, head_dim, "dense_prefill");
  if (rc != NVK_OK) return rc;
  if (batch == 0 || total_q == 0 || max_q_len == 0) return NVK_OK;
  if (total_kv <= 0 || !key || !value || !cu_seqlens_q || !cu_seqlens_kv)
    return fail(NVK_ERR_INVALID_ARGUMENT, "dense_prefill: null pointer or no keys");
  CUtensorMap qm, km, vm;
  if ((rc = kv_tensor_map(&qm, query, total_q, num_heads, kRows)) != NVK_OK) return rc;
  if ((rc = kv_tensor_map(&km, key, total_kv, num_kv_heads, kKeys)) != NVK_OK) return rc;
  if ((rc = kv_tensor_map(&vm, value, total_kv, num_kv_heads, kKeys)) != NVK_OK) return rc;
  PrefillArgs a{};
  a.out = static_cast<__nv_bfloat16*>(out);
  a.block_tables = nullptr;
  a.cu_q = cu_seqlens_q;
  a.kv_lens = nullptr;
  a.cu_kv = cu_seqlens_kv;
  a.err = error_word;
  a.bt_stride = 0;
  a.num_blocks = 0;
  a.num_heads = num_heads;
  a.qpk = num_heads / num_kv_heads;
  a.paged = 0;
  a.batch = batch;
  a.scale_log2 = scale * 1.4426950408889634f;
  return launch_prefill(qm, km, vm, a, max_q_len, reinterpret_cast<cudaStream_t>(stream));
}
