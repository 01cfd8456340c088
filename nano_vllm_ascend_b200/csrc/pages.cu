// Pages (blocks) of a pool: copies from block to block in every layer, clearing,
// and the block tables of pages that moved.
//
// A pool is one or two tensors [layers, num_blocks, block], of any type: a
// block of a layer is block_bytes contiguous bytes. Bound by HBM: each byte is
// read and written once.
// 45 blocks of 128 tokens of a bf16 pool (28 layers of 8 heads) copied and three
// cleared, 1.36 GB, with the tables of 32 sequences: 231 us (0.90 of the
// measured copy rate); by loads and stores, 16 bytes a thread, 285. One block of
// an 8-bit pool of 28 layers, 14.8 MB: 4.9 us with the tables, the kernels'
// latency. Pieces of 4 to 32 KB, 1 to 12 warps and 2 to 4 pieces ahead all ran
// in 230 to 233 us.
#include "host_common.h"
#include "nvk_common.cuh"

namespace nvk {
namespace pages {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = 4;            // of a copying block, one of which an SM holds
constexpr int kPieceBytes = 8192;
constexpr int kStages = 6;           // pieces a warp has room for
constexpr int kAhead = 3;            // of which so many are on their way in

struct CopyArgs {
  uint8_t* base[2];
  const int2* pairs;
  int64_t block_bytes, layer_bytes, items;
  int num_blocks, layers, tensors, parts;
  int* err;
};
struct CopySmem {
  alignas(128) uint8_t ring[kWarps][kStages][kPieceBytes];
  uint64_t full[kWarps][kStages];
};

// A warp takes every n-th piece of the blocks, by bulk copies global -> shared
// -> global through a ring of its own: three pieces on their way in while
// earlier ones go out. The lanes work out 32 pieces at a time, lane 0 copies.
__global__ void __launch_bounds__(32 * kWarps) copy_kernel(const CopyArgs a) {
  extern __shared__ __align__(128) uint8_t smem_raw[];
  CopySmem& sm = *reinterpret_cast<CopySmem*>(smem_raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (lane == 0) {
    for (int s = 0; s < kStages; ++s) mbar_init(&sm.full[warp][s], 1);
    fence_mbar_init();
  }
  __syncwarp();
  pdl_launch_dependents();
  pdl_wait();
  const int64_t step = static_cast<int64_t>(gridDim.x) * kWarps, begin = static_cast<int64_t>(blockIdx.x) * kWarps + warp;
  const int64_t mine = a.items > begin ? (a.items - begin + step - 1) / step : 0;
  // What lane i knows of the batch's piece i: its places (`from` 0: zeros; `to` 0: nothing to do) and size.
  uint64_t from = 0, to = 0;
  int bytes = 0;
  auto look_up = [&](int64_t k) {
    from = to = 0;
    if (k + lane >= mine) return;
    const int64_t w = begin + (k + lane) * step;
    const int64_t block = w / a.parts, lt = static_cast<int64_t>(a.layers) * a.tensors, pair = block / lt;
    const int part = static_cast<int>(w - block * a.parts), rest = static_cast<int>(block - pair * lt);
    const int tensor = rest / a.layers, layer = rest - tensor * a.layers;
    const int2 p = a.pairs[pair];
    if (p.y == -1) return;
    if (p.x < -1 || p.x >= a.num_blocks || p.y < 0 || p.y >= a.num_blocks) {
      if (a.err) atomicOr(a.err, kErrBadBlockId);
      return;
    }
    if (p.x == p.y) return;
    const int64_t at = layer * a.layer_bytes + static_cast<int64_t>(part) * kPieceBytes;
    const uint64_t base = reinterpret_cast<uint64_t>(tensor ? a.base[1] : a.base[0]) + at;
    bytes = static_cast<int>(min(static_cast<int64_t>(kPieceBytes), a.block_bytes - static_cast<int64_t>(part) * kPieceBytes));
    from = p.x < 0 ? 0 : base + p.x * a.block_bytes;
    to = base + p.y * a.block_bytes;
  };
  uint64_t dst[kStages] = {};  // lane 0's, with the sizes, of the pieces in the ring
  int size[kStages] = {};
  int loaded = 0, stored = 0;
  bool ok = true;
  for (int64_t k = 0; ok && (k < mine || stored < loaded);) {
    // One turn of the ring a pass, so that the stage is a constant.
#pragma unroll
    for (int s = 0; s < kStages; ++s) {
      // the next piece that is copied, into stage s; zeros are written on the way
      bool found = false;
      uint64_t f = 0, t = 0;
      int n = 0;
      while (!found && k < mine) {
        if ((k & 31) == 0) look_up(k);
        const int i = static_cast<int>(k & 31);
        f = __shfl_sync(0xffffffffu, from, i);
        t = __shfl_sync(0xffffffffu, to, i);
        n = __shfl_sync(0xffffffffu, bytes, i);
        ++k;
        if (t && !f)
          for (int j = lane; j < n / 16; j += 32) reinterpret_cast<uint4*>(t)[j] = make_uint4(0, 0, 0, 0);
        found = t && f;
      }
      if (found) {
        if (lane == 0) {
          bulk_wait_read<kStages - kAhead - 1>();  // the stage's last piece is out
          mbar_arrive_expect_tx(&sm.full[warp][s], n);
          bulk_load(sm.ring[warp][s], reinterpret_cast<const void*>(f), n, &sm.full[warp][s]);
        }
        dst[s] = t;
        size[s] = n;
        ++loaded;
      }
      // the piece kAhead before it goes out
      if (found ? loaded - stored > kAhead : stored < loaded) {
        constexpr int kBack = kStages - kAhead;
        const int o = (s + kBack) % kStages;
        if (found) {
          if (lane == 0) {
            if (!mbar_wait(&sm.full[warp][o], (stored / kStages) & 1)) {
              ok = false;
            } else {
              bulk_store(reinterpret_cast<void*>(dst[o]), sm.ring[warp][o], size[o]);
              bulk_commit();
            }
          }
          ++stored;
        } else {  // no further piece: what is left, in order
          for (; stored < loaded; ++stored) {
            if (lane == 0) {
              const int q = stored % kStages;
              uint64_t d = 0;
              int z = 0;
#pragma unroll
              for (int e = 0; e < kStages; ++e)
                if (e == q) d = dst[e], z = size[e];
              if (!mbar_wait(&sm.full[warp][q], (stored / kStages) & 1)) {
                ok = false;
              } else {
                bulk_store(reinterpret_cast<void*>(d), sm.ring[warp][q], z);
                bulk_commit();
              }
            }
          }
        }
      }
      ok = __shfl_sync(0xffffffffu, ok, 0);
      if (!ok || (k >= mine && stored == loaded)) break;
    }
  }
  if (lane == 0) {
    if (!ok) {
      if (a.err) atomicOr(a.err, kErrWaitTimeout);
      for (; stored < loaded; ++stored) (void)mbar_wait(&sm.full[warp][stored % kStages], (stored / kStages) & 1);
    }
    bulk_wait_all();
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

int sm_count() {
  int sms = 148, dev = 0;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms;
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
  a.num_blocks = num_blocks;
  a.layers = num_layers;
  a.tensors = pool2 ? 2 : 1;
  const int64_t parts = (block_bytes + kPieceBytes - 1) / kPieceBytes;
  if (parts > (int64_t(1) << 30)) return fail(NVK_ERR_UNSUPPORTED, "%s: blocks of %lld bytes", who, (long long)block_bytes);
  a.parts = static_cast<int>(parts);
  a.err = error_word;
  a.items = static_cast<int64_t>(num_pairs) * num_layers * a.tensors * parts;
  int rc = ensure_dynamic_smem(reinterpret_cast<const void*>(&copy_kernel), sizeof(CopySmem));
  if (rc != NVK_OK) return rc;
  const int64_t want = (a.items + kWarps - 1) / kWarps, sms = sm_count();
  return check_cuda(launch_pdl(copy_kernel, dim3(static_cast<unsigned>(want < sms ? want : sms)), dim3(32 * kWarps),
                               sizeof(CopySmem), reinterpret_cast<cudaStream_t>(stream), a),
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
  const int64_t most = int64_t(sm_count()) * 8;
  return check_cuda(launch_pdl(remap_kernel, dim3(static_cast<unsigned>(want < most ? want : most)),
                               dim3(kThreads), 0, reinterpret_cast<cudaStream_t>(stream), block_tables, row_stride,
                               num_rows, width, map, num_blocks, error_word),
                    "remap_blocks launch");
}
