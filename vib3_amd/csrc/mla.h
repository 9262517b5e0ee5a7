// mla.h — what the latent-attention kernels share: element types and the paged cache's addressing.
#pragma once

#include "common.h"
#include "kernels.h"

namespace vib3 {

// A 16-bit element type by its VIB3_DT_ code.
template <int DT>
__device__ __forceinline__ float to_f32(uint16_t b) {
  return DT == VIB3_DT_F16 ? f16_to_f32(b) : bf16_to_f32(b);
}

template <int DT>
__device__ __forceinline__ uint16_t from_f32(float f) {
  return DT == VIB3_DT_F16 ? f32_to_f16_bits(f) : f32_to_bf16_bits(f);
}

// Eight elements of 16 bytes as f32, and back.
template <int DT>
__device__ __forceinline__ void unpack8(const uint4 v, float* f) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    f[2 * i] = to_f32<DT>((uint16_t)(w[i] & 0xffff));
    f[2 * i + 1] = to_f32<DT>((uint16_t)(w[i] >> 16));
  }
}

template <int DT>
__device__ __forceinline__ uint4 pack8(const float* f) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; i++)
    w[i] = (uint32_t)from_f32<DT>(f[2 * i]) | ((uint32_t)from_f32<DT>(f[2 * i + 1]) << 16);
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Eight elements of a vector of dtype dt (16-byte aligned) as f32.
__device__ __forceinline__ void load8(const void* p, int dt, size_t i, float* f) {
  if (dt == VIB3_DT_F32) {
    const float4 a = *(const float4*)((const float*)p + i), b = *(const float4*)((const float*)p + i + 4);
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
  } else {
    const uint4 v = *(const uint4*)((const uint16_t*)p + i);
    if (dt == VIB3_DT_F16) unpack8<VIB3_DT_F16>(v, f);
    else unpack8<VIB3_DT_BF16>(v, f);
  }
}

// Row of token j of sequence s in the cache (s and j >= 0 checked by the caller), or null where
// the token lies past the block table or on a page that is not resident.
__device__ __forceinline__ const uint16_t* cache_row(const vib3_mla_cache& c, int s, int j) {
  const int page = j / c.page_size;
  if (page >= c.max_pages) return nullptr;
  const int id = c.block_table[(size_t)s * c.max_pages + page];
  if ((unsigned)id >= (unsigned)c.num_pages) return nullptr;
  return (const uint16_t*)c.pool + (int64_t)id * c.page_stride + (int64_t)(j - page * c.page_size) * c.row_stride;
}

// Cached tokens that a row of lens[r] = n sees at most: the block table's capacity bounds n.
__device__ __forceinline__ int clamp_len(const vib3_mla_cache& c, int n) {
  const int64_t cap = (int64_t)c.max_pages * c.page_size;
  return n <= 0 ? 0 : n > cap ? (int)cap : n;
}

// Host checks shared by the launchers.
inline bool mla_aligned(const void* p) { return p && ((uintptr_t)p & 15) == 0; }
inline bool mla_stride(int64_t s) { return s % 8 == 0; }
inline bool mla_dtype(int dt) { return dt == VIB3_DT_F16 || dt == VIB3_DT_BF16; }

inline int check_cache(const vib3_mla_cache& c) {
  if (!mla_dtype(c.dtype) || (c.rank != 256 && c.rank != 512) || (c.rope != 32 && c.rope != 64))
    return VIB3_ERR_UNSUPPORTED;
  if (c.num_pages < 0 || c.page_size < 1 || c.page_size > 65536 || c.num_seqs < 0 || c.max_pages < 0)
    return VIB3_ERR_BAD_COUNT;
  if (c.num_pages && !mla_aligned(c.pool)) return VIB3_ERR_BAD_POINTER;
  if (c.num_seqs && c.max_pages && !c.block_table) return VIB3_ERR_BAD_POINTER;
  if (!mla_stride(c.page_stride) || !mla_stride(c.row_stride)) return VIB3_ERR_BAD_POINTER;
  if (c.row_stride < c.rank + c.rope || c.page_stride < 0) return VIB3_ERR_BAD_COUNT;
  return 0;
}

}  // namespace vib3
