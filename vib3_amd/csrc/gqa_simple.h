// gqa_simple.h — attention of one query head by one wave, token after token, in f32.
#pragma once

#include "gqa.h"

namespace vib3 {

template <int DT, int D>
__device__ void attend_simple(const vib3_gqa_cache& c, int seq, int pos, int kv_head, const uint16_t* q, float scale, int window,
                              int sinks, uint16_t* out) {
  constexpr int E = D / 64;
  const int lane = lane_id();
  float x[E], o[E] = {}, m = -__builtin_huge_valf(), l = 0.0f;
#pragma unroll
  for (int e = 0; e < E; e++) x[e] = to_f32<DT>(q[lane * E + e]);
  const float factor = exponent_scale(scale);
  const int start = window_start(pos, window);
  for (int j = start > 0 && sinks > 0 ? 0 : start; j <= pos; j++) {
    if (j >= sinks && j < start) j = start;
    const int64_t at = gqa_token(c, seq, j);
    if (at < 0) continue;
    const uint16_t* k = (const uint16_t*)c.keys + at + kv_head * c.head_stride + lane * E;
    const uint16_t* v = (const uint16_t*)c.values + at + kv_head * c.head_stride + lane * E;
    float s = 0.0f;
#pragma unroll
    for (int e = 0; e < E; e++) s = __builtin_fmaf(x[e], to_f32<DT>(k[e]), s);
    s = scale < 0.0f ? -wave_sum(s) : wave_sum(s);
    const float top = fmaxf(m, s), ref = top == -__builtin_huge_valf() ? 0.0f : top;
    const float f = exp2f((m - ref) * factor), p = exp2f((s - ref) * factor);
    m = top;
    l = l * f + p;
#pragma unroll
    for (int e = 0; e < E; e++) o[e] = o[e] * f + p * to_f32<DT>(v[e]);
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
  for (int e = 0; e < E; e++) out[lane * E + e] = from_f32<DT>(l == 0.0f ? 0.0f : o[e] * inv);
}

}  // namespace vib3
