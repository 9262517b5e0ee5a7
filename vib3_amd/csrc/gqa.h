// gqa.h — what the grouped-query attention kernels share: the paged cache's addressing, what a query sees, the host's checks.
#pragma once

#include "mla.h"

namespace vib3 {

// Offset of token j of sequence s (both checked by the caller) from the pools' start, in elements, or -1 where the token lies past the
// block table or on a page that is not resident.
__device__ __forceinline__ int64_t gqa_token(const vib3_gqa_cache& c, int s, int j) {
  const int page = j / c.page_size;
  if (page >= c.max_pages) return -1;
  const int id = c.block_table[(size_t)s * c.max_pages + page];
  if ((unsigned)id >= (unsigned)c.num_pages) return -1;
  return (int64_t)id * c.page_stride + (int64_t)(j - page * c.page_size) * c.token_stride;
}

// Cached tokens of a sequence whose length is given as n: the block table's capacity bounds it (and 2^31 - 2^12, so that a token's
// number plus a tile's width stays an int).
__device__ __forceinline__ int gqa_len(const vib3_gqa_cache& c, int n) {
  const int64_t cap = min((int64_t)c.max_pages * c.page_size, (int64_t)0x7ffff000);
  return n <= 0 ? 0 : n > cap ? (int)cap : n;
}

// The first token of the window of position p.
__device__ __forceinline__ int window_start(int p, int window) { return window > 0 && p >= window ? p - window + 1 : 0; }

// Whether eight 16-bit elements are all finite.
template <int DT>
__device__ __forceinline__ bool all_finite(uint4 v) {
  return finite_only<DT>(v.x) == v.x && finite_only<DT>(v.y) == v.y && finite_only<DT>(v.z) == v.z && finite_only<DT>(v.w) == v.w;
}

// Host checks shared by the launchers.
inline int check_gqa_cache(const vib3_gqa_cache& c) {
  if (!mla_dtype(c.dtype) || (c.dim != 64 && c.dim != 128 && c.dim != 256)) return VIB3_ERR_UNSUPPORTED;
  if (c.num_pages < 0 || c.page_size < 1 || c.page_size > 65536 || c.num_seqs < 0 || c.max_pages < 0 || c.kv_heads < 1 ||
      c.kv_heads > 1024)
    return VIB3_ERR_BAD_COUNT;
  if (c.num_pages && (!mla_aligned(c.keys) || !mla_aligned(c.values))) return VIB3_ERR_BAD_POINTER;
  if (c.num_seqs && c.max_pages && !c.block_table) return VIB3_ERR_BAD_POINTER;
  if (!mla_stride(c.page_stride) || !mla_stride(c.token_stride) || !mla_stride(c.head_stride)) return VIB3_ERR_BAD_POINTER;
  if (c.page_stride < 0 || (c.page_size > 1 && c.token_stride < c.dim) || (c.kv_heads > 1 && c.head_stride < c.dim))
    return VIB3_ERR_BAD_COUNT;
  return 0;
}

inline bool gqa_heads(int heads, int kv_heads) { return heads >= 1 && heads <= 1024 && heads % kv_heads == 0; }

}  // namespace vib3
