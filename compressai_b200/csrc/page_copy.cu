// Pages of a cache copied within their pools: what a fork, a compaction of the pool or a spilled prefix needs.
//
// All pools of all layers share page ids, so one launch copies page src[i] to dst[i] in each of them. Moved bytes and
// nothing else: a block takes 16 KB of one page of one pool, four 16-byte loads a thread in flight.
#include "common.cuh"

namespace vq2 {
namespace {

constexpr int kPools = 128;              // of one launch: 2 KB of arguments
constexpr int kThreads = 256, kLoads = 4, kTile = kThreads * kLoads;   // 16-byte pieces of a block

struct CopyArgs {
  struct {
    uint4* base;
    uint32_t vecs;    // 16-byte pieces of a page
    uint32_t first;   // blocks of a pair before this pool's
  } pool[kPools];
  const int32_t *src, *dst;
  int n_pools, pages;
  uint32_t blocks;    // of a pair
};

__global__ void __launch_bounds__(kThreads) copy_pages_kernel(const __grid_constant__ CopyArgs a) {
  pdl_wait();
  pdl_trigger();
  const uint32_t i = blockIdx.x / a.blocks, part = blockIdx.x - i * a.blocks;
  const int src = a.src[i], dst = a.dst[i];
  if (src < 0 || src >= a.pages || dst < 0 || dst >= a.pages || src == dst) return;
  int p = 0;   // the last pool that starts at or before this block
  for (int step = kPools / 2; step; step >>= 1)
    if (p + step < a.n_pools && a.pool[p + step].first <= part) p += step;
  const uint32_t vecs = a.pool[p].vecs, at = (part - a.pool[p].first) * kTile + threadIdx.x;
  const uint4* from = a.pool[p].base + (int64_t)src * vecs;
  uint4* to = a.pool[p].base + (int64_t)dst * vecs;
  uint4 x[kLoads];
#pragma unroll
  for (int k = 0; k < kLoads; ++k)
    if (at + k * kThreads < vecs) x[k] = from[at + k * kThreads];
#pragma unroll
  for (int k = 0; k < kLoads; ++k)
    if (at + k * kThreads < vecs) to[at + k * kThreads] = x[k];
}

}  // namespace
}  // namespace vq2

using namespace vq2;

extern "C" int vq2_copy_pages(const vq2_page_pool* pools, int64_t n_pools, int64_t pages, const int32_t* src,
                              const int32_t* dst, int64_t n, void* stream) {
  if (n_pools < 0 || n < 0 || (n_pools && !pools) || (n && (!src || !dst))) return VQ2_ERR_ARG;
  if (pages < 1 || pages > 0x7fffffff || n > 0x7fffffff) return VQ2_ERR_SHAPE;
  for (int64_t p = 0; p < n_pools; ++p) {
    if (!pools[p].base) return VQ2_ERR_ARG;
    if (!aligned(pools[p].base, 16) || pools[p].page_bytes % 16) return VQ2_ERR_ALIGN;
    if (pools[p].page_bytes < 0 || pools[p].page_bytes > int64_t(1) << 30) return VQ2_ERR_SHAPE;
  }
  for (int64_t p0 = 0; p0 < n_pools; p0 += kPools) {
    CopyArgs a = {};
    int64_t blocks = 0;
    for (int64_t p = p0; p < n_pools && p < p0 + kPools; ++p) {
      if (pools[p].page_bytes == 0) continue;
      auto& to = a.pool[a.n_pools++];
      to.base = static_cast<uint4*>(pools[p].base);
      to.vecs = (uint32_t)(pools[p].page_bytes / 16);
      to.first = (uint32_t)blocks;
      blocks += (to.vecs + kTile - 1) / kTile;   // 2^23 a launch at most
    }
    if (!blocks) continue;
    a.pages = (int)pages;
    a.blocks = (uint32_t)blocks;
    const int64_t most = 0x7fffffff / blocks;   // pairs of one launch
    for (int64_t i = 0; i < n; i += most) {
      a.src = src + i;
      a.dst = dst + i;
      const int64_t pairs = n - i < most ? n - i : most;
      const int s = launch_kernel(copy_pages_kernel, dim3((unsigned)(pairs * blocks)), dim3(kThreads), 0,
                                  static_cast<cudaStream_t>(stream), a);
      if (s != VQ2_OK) return s;
    }
  }
  return VQ2_OK;
}
