// Pages (blocks) of a pool: copies from block to block in every layer, clearing,
// and the block tables of pages that moved.
//
// A pool is one or two tensors [layers, num_blocks, block], of any type: a
// block of a layer is block_bytes contiguous bytes. Bound by HBM: each byte is
// read and written once.
#include "host_common.h"
#include "nvk_common.cuh"

namespace nvk {
namespace pages {
namespace {

constexpr int kThreads = 256;

struct CopyArgs {
  uint8_t* base[2];
  const int2* pairs;
  int64_t block_bytes, layer_bytes;
  int num_pairs, num_blocks, layers, tensors, parts;
  int64_t part_bytes;
  int* err;
};

// A block takes part x of pair y's copy in layer z of a tensor.
__global__ void __launch_bounds__(kThreads) copy_kernel(const CopyArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  const int64_t items = static_cast<int64_t>(a.num_pairs) * a.layers * a.tensors * a.parts;
  for (int64_t w = blockIdx.x; w < items; w += gridDim.x) {
    const int part = static_cast<int>(w % a.parts);
    int64_t rest = w / a.parts;
    const int layer = static_cast<int>(rest % a.layers);
    rest /= a.layers;
    const int tensor = static_cast<int>(rest % a.tensors);
    const int2 p = a.pairs[rest / a.tensors];
    if (p.y == -1) continue;
    if (p.x < -1 || p.x >= a.num_blocks || p.y < 0 || p.y >= a.num_blocks) {
      if (threadIdx.x == 0 && a.err) atomicOr(a.err, kErrBadBlockId);
      continue;
    }
    if (p.x == p.y) continue;
    uint8_t* at = a.base[tensor] + layer * a.layer_bytes + part * a.part_bytes;
    const int64_t bytes = min(a.part_bytes, a.block_bytes - part * a.part_bytes);
    const uint4* src = reinterpret_cast<const uint4*>(at + max(p.x, 0) * a.block_bytes);
    uint4* dst = reinterpret_cast<uint4*>(at + p.y * a.block_bytes);
    for (int64_t i = threadIdx.x; i < bytes / 16; i += kThreads)
      dst[i] = p.x < 0 ? make_uint4(0, 0, 0, 0) : src[i];
  }
}

__global__ void __launch_bounds__(kThreads) remap_kernel(int32_t* tables, int64_t stride, int64_t rows, int width,
                                                         const int32_t* map, int num_blocks, int* err) {
  pdl_wait();
  const int64_t items = rows * width;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < items;
       i += static_cast<int64_t>(gridDim.x) * kThreads) {
    int32_t* at = tables + i / width * stride + i % width;
    const int b = *at;
    const int to = b >= 0 && b < num_blocks ? map[b] : -1;
    if (to < 0 || to >= num_blocks) {
      if (err) atomicOr(err, kErrBadBlockId);
    } else {
      *at = to;
    }
  }
}

}  // namespace
}  // namespace pages
}  // namespace nvk

extern "C" int nvk_copy_blocks(void* pool, void* pool2, int num_layers, int num_blocks, int64_t block_bytes,
                               const int32_t* pairs, int num_pairs, int* error_word, nvk_stream_t stream) {
  using namespace nvk;
  using namespace nvk::pages;
  const char* who = "copy_blocks";
  if (num_layers <= 0 || num_blocks <= 0 || block_bytes <= 0 || num_pairs < 0)
    return fail(NVK_ERR_INVALID_ARGUMENT, "%s: bad sizes (layers=%d blocks=%d block_bytes=%lld pairs=%d)", who,
                num_layers, num_blocks, (long long)block_bytes, num_pairs);
  if (block_bytes % 16)
    return fail(NVK_ERR_UNSUPPORTED, "%s: blocks of %lld bytes (multiples of 16 only)", who, (long long)block_bytes);
  if (num_pairs == 0) return NVK_OK;
  if (!pool || !pairs) return fail(NVK_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
  if (!aligned16(pool) || !aligned16(pool2) || (reinterpret_cast<uintptr_t>(pairs) & 7u))
    return fail(NVK_ERR_INVALID_ARGUMENT, "%s: pools must be 16-byte aligned, pairs 8-byte aligned", who);
  CopyArgs a;
  a.base[0] = static_cast<uint8_t*>(pool);
  a.base[1] = static_cast<uint8_t*>(pool2);
  a.pairs = reinterpret_cast<const int2*>(pairs);
  a.block_bytes = block_bytes;
  a.layer_bytes = block_bytes * num_blocks;
  a.num_pairs = num_pairs;
  a.num_blocks = num_blocks;
  a.layers = num_layers;
  a.tensors = pool2 ? 2 : 1;
  a.part_bytes = 16384;
  const int64_t parts = (block_bytes + a.part_bytes - 1) / a.part_bytes;
  if (parts > (int64_t(1) << 30)) return fail(NVK_ERR_UNSUPPORTED, "%s: blocks of %lld bytes", who, (long long)block_bytes);
  a.parts = static_cast<int>(parts);
  a.err = error_word;
  const int64_t items = static_cast<int64_t>(num_pairs) * num_layers * a.tensors * parts;
  return check_cuda(launch_pdl(copy_kernel, dim3(static_cast<unsigned>(items < 148 * 8 ? items : 148 * 8)),
                               dim3(kThreads), 0, reinterpret_cast<cudaStream_t>(stream), a),
                    "copy_blocks launch");
}

extern "C" int nvk_remap_blocks(int32_t* block_tables, int64_t row_stride, int64_t num_rows, int width,
                                const int32_t* map, int num_blocks, int* error_word, nvk_stream_t stream) {
  using namespace nvk;
  using namespace nvk::pages;
  const char* who = "remap_blocks";
  if (num_rows < 0 || width < 0 || num_blocks <= 0 || (num_rows > 1 && row_stride < width))
    return fail(NVK_ERR_INVALID_ARGUMENT, "%s: bad sizes (rows=%lld width=%d stride=%lld blocks=%d)", who,
                (long long)num_rows, width, (long long)row_stride, num_blocks);
  if (num_rows == 0 || width == 0) return NVK_OK;
  if (!block_tables || !map) return fail(NVK_ERR_INVALID_ARGUMENT, "%s: null pointer", who);
  const int64_t want = (num_rows * width + kThreads - 1) / kThreads;
  return check_cuda(launch_pdl(remap_kernel, dim3(static_cast<unsigned>(want < 148 * 8 ? want : 148 * 8)),
                               dim3(kThreads), 0, reinterpret_cast<cudaStream_t>(stream), block_tables, row_stride,
                               num_rows, width, map, num_blocks, error_word),
                    "remap_blocks launch");
}
