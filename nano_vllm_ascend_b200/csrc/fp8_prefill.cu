// Causal prefill attention over the 8-bit KV pool (cached prefix and the rows
// appended this step). The kernel body, with its design, is in
// prefill_core.cuh; the pool's format is in fp8_kv.cuh.
//
// Tensor-bound by its operations (4 * 128 a visible pair and head), in practice
// by the chains of a tile: 97.2 us for 32 requests of 256 tokens over 768 cached
// ones (16 heads on 8, blocks of 128; 60.2 GFLOP, 619 TF/s, tensor pipe 37 % of
// its cycles), where the 4-bit kernel takes 80 to 82 and the bf16 one 71.5. The
// decoders turn two codes a conversion (2 cycles a warp instruction, measured)
// and a tile's 32768 codes pass four warps, beside 8 of softmax that take an
// exponent a unit. Ways that were built and measured for the same work: fp16 or
// bf16 products of code and exponent by the decoders 106 to 158 us (spills, and
// the wider range of bf16 costs P three bits); codes brought in by bulk copies, by
// the decoding or a further warp, 96 to 107; eight decoding warps of 20 98 to
// 105; both operands' registers double 98 to 115; each unit asked into L2 two to
// five tiles ahead 98 to 101; with one stream, the idle softmax warpgroup as
// second decoder 25.5 instead of 24.6 for five ragged requests. Those five (up to
// 300 tokens over up to 1000, 9 heads on 3) are bound by latency: each walks up
// to 9 tiles of 2.0 us, whatever their 1.7 us of operations.
#include "prefill_core.cuh"

#include <atomic>

namespace nvk {
using namespace prefill;
namespace {

__global__ void __launch_bounds__(kThreadsDecoding, 1) fp8_prefill_kernel(const __grid_constant__ CUtensorMap qmap,
                                                                          const PrefillArgs a) {
  prefill_body<kHeldFp8>(qmap, qmap, qmap, a);
}

__global__ void __launch_bounds__(kThreadsDecoding, 1) fp8_prefill_parts_kernel(const __grid_constant__ CUtensorMap qmap,
                                                                                const PrefillArgs a) {
  prefill_body<kHeldFp8, true>(qmap, qmap, qmap, a);
}

constexpr size_t kSmem = sizeof(PrefillSmem) + 1024;

struct ClusterLaunch {
  cudaLaunchAttribute attr[2];
  cudaLaunchConfig_t cfg{};
  ClusterLaunch(int clusters, int ranks, cudaStream_t stream) {
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim = {static_cast<unsigned>(ranks), 1, 1};
    cfg.gridDim = dim3(clusters * ranks);
    cfg.blockDim = dim3(kThreadsDecoding);
    cfg.dynamicSmemBytes = kSmem;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
  }
};

// Clusters of `ranks` CTAs that run at once on device `dev`; asked once.
int clusters_at_once(int dev, int ranks) {
  constexpr int kDevices = 64;
  static std::atomic<int> known[kDevices][kMostParts + 1];
  if (dev < 0 || dev >= kDevices) return 0;
  int n = known[dev][ranks].load(std::memory_order_relaxed);
  if (n == 0) {
    ClusterLaunch at(1, ranks, nullptr);
    if (cudaOccupancyMaxActiveClusters(&n, fp8_prefill_parts_kernel, &at.cfg) != cudaSuccess) n = 0;
    if (n <= 0) {
      cudaGetLastError();
      n = -1;
    }
    known[dev][ranks].store(n, std::memory_order_relaxed);
  }
  return n;
}

}  // namespace
}  // namespace nvk

extern "C" int nvk_fp8_paged_prefill(void* out, const void* query, const void* kv_cache, int num_blocks,
                                     int block_size, const int32_t* block_tables, int block_table_stride,
                                     int max_blocks_per_seq, const int32_t* cu_seqlens_q, const int32_t* kv_lens,
                                     int batch, int total_q, int max_q_len, int num_heads, int num_kv_heads,
                                     int head_dim, float scale, int* error_word,
                                     nvk_stream_t stream) {
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
  a.paged = 1;
  a.batch = batch;
  a.qtiles = (max_q_len + kRows - 1) / kRows;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.pool = static_cast<const uint8_t*>(kv_cache);
  a.kvh = num_kv_heads;
  a.upb_log2 = fp8::units_log2(block_size);
  a.max_blocks = max_blocks_per_seq;
  a.total_q = total_q;
  a.out_scale = 1.f;
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  // Two heads an item share the tiles of a KV head; where one head an item leaves none of the SMs a second one, that
  // (512 queries over 1024 keys, 16 heads on 8: 25.1 us with two heads an item, 21 with one); where it leaves half of
  // the SMs or more without an item, its keys over a cluster's CTAs, as many as run at once (see kSavedTiles). The host
  // knows the table's width, not the lengths: a short context under a wide table launches CTAs that only meet at the
  // cluster's barriers (up to 512 keys in a table of 40960 0.7 to 1.6 us more, 8.0 -> 9.4 us for four prompts of 100 queries), and
  // how an item is divided, and with it the last bits, follow from the width and the number of items.
  const int64_t alone = static_cast<int64_t>(a.qtiles) * num_heads * batch;
  a.paired = a.qpk % 2 == 0 && alone > sms;
  const int64_t items = a.paired ? alone / kStreams : alone;
  if (items > (int64_t(1) << 30))
    return fail(NVK_ERR_UNSUPPORTED, "%s: %lld work items above the kernel's range", who, (long long)items);
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int64_t most_tiles = (static_cast<int64_t>(max_blocks_per_seq) * block_size + kKeys - 1) / kKeys;
  for (int ranks = 2 * items <= sms ? kMostParts : 1; ranks > 1; --ranks) {
    const int64_t per = (most_tiles + ranks - 1) / ranks;
    if (most_tiles - per < kSavedTiles) break;
    if (items * ranks > sms) continue;
    rc = ensure_dynamic_smem(reinterpret_cast<const void*>(&fp8_prefill_parts_kernel), kSmem);
    if (rc != NVK_OK) return rc;
    if (items > clusters_at_once(dev, ranks)) continue;
    ClusterLaunch at(static_cast<int>(items), static_cast<int>((most_tiles + per - 1) / per), st);
    return check_cuda(cudaLaunchKernelEx(&at.cfg, fp8_prefill_parts_kernel, qm, a), "fp8_paged_prefill launch");
  }
  if ((rc = ensure_dynamic_smem(reinterpret_cast<const void*>(&fp8_prefill_kernel), kSmem)) != NVK_OK) return rc;
  const int grid = static_cast<int>(items < sms ? items : sms);
  return check_cuda(launch_pdl(fp8_prefill_kernel, dim3(grid), dim3(kThreadsDecoding), kSmem, st, qm, a),
                    "fp8_paged_prefill launch");
}
