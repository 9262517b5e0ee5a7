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

// Cached tokens that a row of lens[r] = n sees at most: the block table's capacity bounds n (and 2^31 - 128, so
// that a token's number plus a tile's width stays an int).
__device__ __forceinline__ int clamp_len(const vib3_mla_cache& c, int n) {
  const int64_t cap = min((int64_t)c.max_pages * c.page_size, (int64_t)0x7fffff80);
  return n <= 0 ? 0 : n > cap ? (int)cap : n;
}

// The factor of scores as exponents of two, without its sign: that goes into the queries (sign_flip) or the scores. A scale of 0
// becomes the smallest number, so that an empty maximum (-infinity) times it stays what it is, and one past f32's range the largest.
__device__ __forceinline__ float exponent_scale(float scale) {
  return fminf(fmaxf(__builtin_fabsf(scale) * 1.44269504088896341f, 1.17549435e-38f), 3.40282347e+38f);
}
// Exponents are formed as fma(score, scale, -m * scale), one operation, with the rounding of m * scale in all that a reference m
// serves: 2^-17 for products up to this. Beyond (by 2^27 it would leave f16's range), m is taken off the scores first.
constexpr float kFarExponent = 256.0f;
__device__ __forceinline__ uint32_t sign_flip(float scale) { return scale < 0.0f ? 0x80008000u : 0u; }

// Probabilities are formed as 2^(kProbShift + (score - reference) in log2 units) and rounded to 16 bits for the matrix cores, sums are
// divided by the sum of the same. The reference of a row follows its running maximum only where that grew by more than kLag: sums are
// seldom rescaled, and what lies up to 2^kLag above the reference is as exact as what lies below. f16 has steps down to 2^-24 only
// (below 2^-14 they no longer shrink with the number), and up to 2^16: with 2^(11 + 4) as the largest probability, those down to
// 2^-25 of the reference keep all of their bits, and no other is off by more than 2^-36 of it. (Without the shift one key 18 nats above
// 8192 others, which hold the values, took them to 0.) bf16 has f32's range.
template <int DT>
constexpr float kProbShift = DT == VIB3_DT_F16 ? 11.0f : 0.0f;
template <int DT>
constexpr float kLag = DT == VIB3_DT_F16 ? 4.0f : 8.0f;

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

namespace vib3 {

// ------------------------------------------------------------------------- matrix cores
//
// Operand layouts of the 16x16x32 products: lane l holds row (A) or column (B) l % 16 at k = 8 (l / 16) + 0..7; of the
// result, column l % 16 of rows 4 (l / 16) + 0..3.

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

template <int DT>
__device__ __forceinline__ f32x4 mma32(s16x8 a, s16x8 b, f32x4 c) {
  if (DT == VIB3_DT_F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// Two f32 rounded to a pair of 16-bit elements (nearest even).
template <int DT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if (DT == VIB3_DT_F16) return __builtin_bit_cast(uint32_t, h2{(half_t)a, (half_t)b});
  return __builtin_bit_cast(uint32_t, bf16x2{(__bf16)a, (__bf16)b});
}

// Two f32 as pairs of 16-bit elements: each number's rounding and, rounded again, what that left (in bf16 off by at most 2^-16 of
// the number, in f16 by 2^-22 of it or 2^-25). A number that rounds to infinity has no rest.
struct Halves {
  uint32_t hi, lo;
};
template <int DT>
__device__ __forceinline__ Halves split2(float a, float b) {
  const uint32_t hi = pack2<DT>(a, b);
  const float x = a - to_f32<DT>((uint16_t)(hi & 0xffff)), y = b - to_f32<DT>((uint16_t)(hi >> 16));
  return Halves{hi, pack2<DT>(__builtin_isfinite(x) ? x : 0.0f, __builtin_isfinite(y) ? y : 0.0f)};
}

typedef __attribute__((address_space(3))) uint8_t lds_u8;

// 16 bytes a lane from global memory to LDS at base + 16 * lane (base wave-uniform), without passing
// through registers. Written as an instruction because the compiler lets every LDS read wait for every such load in
// flight, also those into another buffer; it has no result register, and it is counted by vmcnt, which the caller waits
// for (wait_lds_loads) before the barrier that publishes the tile. Waits that the compiler places for its own loads only come out
// stricter by it.
__device__ __forceinline__ void load_to_lds16(const void* g, lds_u8* base) {
  const uint32_t at = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(uintptr_t)base);
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(at), "v"(g) : "memory", "m0");
}

// The same with 4 bytes a lane, at base + 4 * lane.
__device__ __forceinline__ void load_to_lds4(const void* g, lds_u8* base) {
  const uint32_t at = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(uintptr_t)base);
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(at), "v"(g) : "memory", "m0");
}

__device__ __forceinline__ void wait_lds_loads() {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

__device__ __forceinline__ s16x8 lds_read16(const lds_u8* p) {
  return *(const __attribute__((address_space(3))) s16x8*)p;
}

__device__ __forceinline__ void lds_write8(lds_u8* p, uint32_t a, uint32_t b) {
  typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
  *(__attribute__((address_space(3))) u32x2*)p = u32x2{a, b};
}

// Transposing read: 16 lanes address 4 rows of 16 elements (lane i: row i / 4, elements 4 (i % 4) + 0..3)
// and lane i receives column i of the 4 rows.
__device__ __forceinline__ s16x4 lds_read_tr(lds_u8* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p);
}

__device__ __forceinline__ s16x8 join(s16x4 a, s16x4 b) {
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

// v as a value that the compiler does not know to be the same each time: what is formed from it is formed where it is used,
// not held in registers over the loop.
__device__ __forceinline__ int fresh(int v) {
  asm volatile("" : "+v"(v));
  return v;
}

}  // namespace vib3
