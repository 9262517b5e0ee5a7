// scan.h — sums over the lanes of a wave, division by a number that a launch fixes, and launches of any number of workgroups.
#pragma once

#include "common.h"

namespace vib3 {

// v of this lane combined with those of the lanes below, by `f`; `none` does nothing there. Lane 63 has all. (All lanes take part.)
template <typename T, typename F>
__device__ __forceinline__ T wave_scan(T v, T none, F f) {
  static_assert(sizeof(T) == 4, "a register a lane");
  const int o = __builtin_bit_cast(int, none);
  auto step = [&](int moved) { v = f(v, __builtin_bit_cast(T, moved)); };
  step(__builtin_amdgcn_update_dpp(o, __builtin_bit_cast(int, v), 0x111, 0xf, 0xf, false));  // from the lane below in a row of 16
  step(__builtin_amdgcn_update_dpp(o, __builtin_bit_cast(int, v), 0x112, 0xf, 0xf, false));  // 2, 4 and 8 below
  step(__builtin_amdgcn_update_dpp(o, __builtin_bit_cast(int, v), 0x114, 0xf, 0xf, false));
  step(__builtin_amdgcn_update_dpp(o, __builtin_bit_cast(int, v), 0x118, 0xf, 0xf, false));
  step(__builtin_amdgcn_update_dpp(o, __builtin_bit_cast(int, v), 0x142, 0xa, 0xf, false));  // lane 15's to the second row, 47's to the last
  step(__builtin_amdgcn_update_dpp(o, __builtin_bit_cast(int, v), 0x143, 0xc, 0xf, false));  // lane 31's to the upper half
  return v;
}

// Sum over the lanes up to this one.
__device__ __forceinline__ int add_up(int v) {
  return wave_scan(v, 0, [](int a, int b) { return a + b; });
}

// t / n for 0 <= t < 2^31: with factor = ceil(2^(31 + shift) / n) and n <= 2^shift, t * factor is above t * 2^(31 + shift) / n by less
// than 2^(31 + shift) / n, which does not reach the next multiple of 2^(31 + shift).
struct Divisor {
  uint32_t factor;
  int shift;
  __device__ __forceinline__ int of(int t) const { return (int)(__umulhi((uint32_t)t << 1, factor) >> shift); }
};
inline Divisor divisor(int n) {
  int shift = 0;
  while ((int64_t)1 << shift < n) shift++;
  return Divisor{(uint32_t)((((uint64_t)1 << (31 + shift)) + (uint64_t)n - 1) / (uint64_t)n), shift};
}

// A grid of at least this many workgroups (up to 2^31). A dimension holds fewer than 2^32 threads, so many workgroups are rows of 2^21;
// those past the number end at once. wide_block: a workgroup's place in it.
inline dim3 wide_grid(int64_t blocks) {
  constexpr int64_t kRow = 1 << 21;
  return blocks <= kRow ? dim3((unsigned)blocks) : dim3((unsigned)kRow, (unsigned)((blocks + kRow - 1) / kRow));
}
__device__ __forceinline__ unsigned wide_block() { return blockIdx.y * gridDim.x + blockIdx.x; }

}  // namespace vib3
