// The paged key/value cache as the kernels see it: argument checks, and how a token finds its
// sequence, its position and its row of the pool. What a caller leaves wrong in device memory (a
// page id outside the pool, a length past the table) reads or writes nothing out of range.
#pragma once
#include <string.h>

#include "common.cuh"

namespace vq2 {

struct PagedKV {
  const void *k, *v;             // [pages, heads, page_size, D] 16-bit or int8
  const float *k_scale, *v_scale;  // int8: [pages, heads, page_size]
  const int32_t* table;          // [seqs, cols] page ids, row stride table_stride
  const int32_t* lens;           // [seqs] tokens in the cache, the new ones among them
  const int32_t* starts;         // [seqs + 1] first new token of each sequence; null: one token each
  int64_t table_stride;
  int32_t pages, heads, page_log2, cols, seqs;
};

inline bool bad_head_size(int64_t D) { return D < 16 || D > 256 || D % 16; }

// Checks what every cache entry point shares and fills `kv`.
inline int paged_kv(PagedKV& kv, const void* k, const void* v, int kv_dtype, const float* k_scale, const float* v_scale,
                    int64_t pages, int64_t heads, int64_t page_size, int64_t D, const int32_t* table,
                    int64_t table_stride, int64_t cols, const int32_t* lens, const int32_t* starts, int64_t seqs) {
  if (!k || !v || (!table && seqs > 0 && cols > 0)) return VQ2_ERR_ARG;   // an empty table may have no address
  if (kv_dtype != VQ2_F16 && kv_dtype != VQ2_BF16 && kv_dtype != VQ2_I8) return VQ2_ERR_DTYPE;
  if ((kv_dtype == VQ2_I8) != (k_scale != nullptr) || (k_scale == nullptr) != (v_scale == nullptr)) return VQ2_ERR_ARG;
  if (page_size < 16 || page_size > 256 || (page_size & (page_size - 1)) || bad_head_size(D)) return VQ2_ERR_SHAPE;
  if (pages < 1 || heads < 1 || heads > 4096 || seqs < 0 || seqs > 0x7ffffff || cols < 0 || table_stride < 0)
    return VQ2_ERR_SHAPE;
  if (pages > 0x7fffffff / page_size || pages * page_size > 0x7fffffff / heads || cols > 0x7fffff00 / page_size)
    return VQ2_ERR_SHAPE;  // a pool's rows and a sequence's positions, and the 255 after them, are counted in 32 bits
  if (!aligned(k, 16) || !aligned(v, 16) || !aligned(k_scale, 16) || !aligned(v_scale, 16)) return VQ2_ERR_ALIGN;
  int l = 4;
  while ((1 << l) < page_size) ++l;
  kv = {k, v, k_scale, v_scale, table, lens, starts, table_stride, (int32_t)pages, (int32_t)heads, l, (int32_t)cols,
        (int32_t)seqs};
  return VQ2_OK;
}

// Sequences whose new tokens end at or before token t. Block-wide (every thread calls it): one
// round trip instead of a search's chain of them.
__device__ __forceinline__ int sequences_before(const PagedKV& kv, int t) {
  int b = 0;
  for (int i = 0; i < kv.seqs; i += blockDim.x) {
    const int j = i + (int)threadIdx.x;
    b += __syncthreads_count(j < kv.seqs && kv.starts[j + 1] <= t);
  }
  return b;
}

// The sequence that new token t belongs to, or -1 (block-wide).
__device__ __forceinline__ int sequence_of(const PagedKV& kv, int t) {
  if (!kv.starts) return t < kv.seqs ? t : -1;
  const int b = sequences_before(kv, t);
  return b < kv.seqs && kv.starts[b] <= t ? b : -1;
}

// Tokens of sequence b in the cache, at most what its table row has room for.
__device__ __forceinline__ int length_of(const PagedKV& kv, int b) {
  return max(0, min(kv.lens[b], kv.cols << kv.page_log2));
}

// First new token and count of new tokens of sequence b.
__device__ __forceinline__ void sequence_rows(const PagedKV& kv, int b, int& first, int& count) {
  first = kv.starts ? kv.starts[b] : b;
  count = kv.starts ? kv.starts[b + 1] - first : 1;
}

// page * page_size + row of position p of sequence b, or -1 where the table has no page for it.
__device__ __forceinline__ int64_t slot_of(const PagedKV& kv, int b, int64_t p) {
  if (p < 0 || (p >> kv.page_log2) >= kv.cols) return -1;
  const int page = kv.table[b * kv.table_stride + (p >> kv.page_log2)];
  if (page < 0 || page >= kv.pages) return -1;
  return ((int64_t)page << kv.page_log2) + (p & ((1 << kv.page_log2) - 1));
}

// Row of the pool ([pages, heads, page_size] flattened) of a slot and head.
__device__ __forceinline__ int64_t pool_row(const PagedKV& kv, int64_t slot, int h) {
  const int64_t page = slot >> kv.page_log2;
  return ((page * kv.heads + h) << kv.page_log2) + (slot & ((1 << kv.page_log2) - 1));
}

}  // namespace vq2
