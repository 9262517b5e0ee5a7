// mla_append.hip — new tokens into the paged latent cache: RMSNorm of the latent, rotation of the
// shared key and of the queries' rotary part, in one launch.
//
// Bound: bytes for prompts (every value read and written once; 6201 tokens of 64 heads, 122 MB, in 28 us: 4.3 TB/s of the 5.0 that
// a large copy reaches), the launch for single tokens (3.2 us on the device, 12 us a call from Python).
// A wave takes one kv row: lane l holds eight neighbouring latent elements (16 bytes; with rank 256 half the lanes), the sum of squares
// is one wave reduction, and the first rope / 2 lanes turn one pair each. A workgroup of the rest takes the heads of one
// token: its first rope / 2 threads form the cosines and sines once (the angle and its reduction in 64 bits: positions reach 10^6
// radians, where f32 angles are off by 0.03) while the queries are on their way, and each thread turns eight pairs, 32 bytes, of
// one head at a time.
#include "mla.h"

namespace vib3 {

// Cosine and sine of p * inv_freq, times g.
__device__ __forceinline__ float2 turn_of(int p, float inv_freq, float g) {
  double t = (double)p * (double)inv_freq * 0.15915494309189535;  // turns
  t -= __builtin_rint(t);
  float s, c;
  sincospif(2.0f * (float)t, &s, &c);
  return make_float2(g * c, g * s);
}

template <int DT>
__global__ __launch_bounds__(256) void k_mla_append(vib3_mla_append a, int kv_blocks) {
  const int tid = (int)threadIdx.x;
  const int rank = a.cache.rank, rope = a.cache.rope, half = rope / 2;
  if ((int)blockIdx.x < kv_blocks) {
    const int t = (int)blockIdx.x * 4 + (tid >> 6), lane = tid & 63;
    if (t >= a.tokens) return;
    const int s = a.seqs[t], p = a.positions[t];
    if ((unsigned)s >= (unsigned)a.cache.num_seqs || p < 0) return;
    const size_t at = (size_t)t * a.kv_stride;
    uint16_t* row = (uint16_t*)cache_row(a.cache, s, p);
    uint16_t* copy = a.kv_out ? (uint16_t*)a.kv_out + (size_t)t * a.kv_out_stride : nullptr;
    // the rotary pair of this lane (lanes past rope / 2 have none)
    const int i0 = a.interleaved ? 2 * lane : lane, i1 = a.interleaved ? 2 * lane + 1 : lane + half;
    float x0 = 0.0f, x1 = 0.0f;
    if (lane < half) {
      x0 = load_act(a.kv, a.kv_dtype, at + rank + i0);
      x1 = load_act(a.kv, a.kv_dtype, at + rank + i1);
    }
    const bool mine = lane * 8 < rank;
    float c[8] = {};
    if (mine) load8(a.kv, a.kv_dtype, at + lane * 8, c);
    if (a.norm_weight) {
      float w[8] = {}, ss = 0.0f;
      if (mine) unpack8<VIB3_DT_F16>(*(const uint4*)((const uint16_t*)a.norm_weight + lane * 8), w);
#pragma unroll
      for (int i = 0; i < 8; i++) ss = __builtin_fmaf(c[i], c[i], ss);
      ss = wave_sum(ss);
      const float inv = 1.0f / sqrtf(ss / (float)rank + a.norm_eps);
#pragma unroll
      for (int i = 0; i < 8; i++) c[i] = c[i] * inv * w[i];
    }
    float2 cs = make_float2(0.0f, 0.0f);
    if (lane < half) cs = turn_of(p, a.inv_freq[lane], a.rope_scale);
    const uint16_t y0 = from_f32<DT>(x0 * cs.x - x1 * cs.y), y1 = from_f32<DT>(x0 * cs.y + x1 * cs.x);
#pragma unroll
    for (int k = 0; k < 2; k++) {
      uint16_t* dst = k ? copy : row;
      if (!dst) continue;
      if (mine) *(uint4*)(dst + lane * 8) = pack8<DT>(c);
      if (lane < half) {
        dst[rank + i0] = y0;
        dst[rank + i1] = y1;
      }
    }
    return;
  }
  // the queries' rotary part
  const int t = (int)blockIdx.x - kv_blocks;
  const int p = a.positions[t];
  if ((unsigned)a.seqs[t] >= (unsigned)a.cache.num_seqs || p < 0) return;
  __shared__ float2 cs[32];
  const int units = half / 8;  // threads on one head
  const int total = a.heads * units;
  const uint16_t* q = (const uint16_t*)a.q_rope + (int64_t)t * a.q_token_stride;
  uint16_t* o = (uint16_t*)a.q_out + (int64_t)t * a.q_out_token_stride;
  // pairs 8 (u % units) .. + 7 of head u / units: two runs of eight elements
  auto first = [&](int u) { return a.interleaved ? 16 * (u % units) : 8 * (u % units); };
  const int second = a.interleaved ? 8 : half;
  uint4 x0, x1;
  auto fetch = [&](int u) {
    const uint16_t* p = q + (int64_t)(u / units) * a.q_head_stride + first(u);
    x0 = *(const uint4*)p;
    x1 = *(const uint4*)(p + second);
  };
  if (tid < total) fetch(tid);
  if (tid < half) cs[tid] = turn_of(p, a.inv_freq[tid], a.rope_scale);
  __syncthreads();
  for (int u = tid; u < total; u += 256) {
    float x[16], y[16];
    unpack8<DT>(x0, x);
    unpack8<DT>(x1, x + 8);
    uint16_t* to = o + (int64_t)(u / units) * a.q_out_head_stride + first(u);
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const float2 w = cs[8 * (u % units) + i];
      if (a.interleaved) {
        y[2 * i] = x[2 * i] * w.x - x[2 * i + 1] * w.y;
        y[2 * i + 1] = x[2 * i] * w.y + x[2 * i + 1] * w.x;
      } else {
        y[i] = x[i] * w.x - x[i + 8] * w.y;
        y[i + 8] = x[i] * w.y + x[i + 8] * w.x;
      }
    }
    if (u + 256 < total) fetch(u + 256);
    *(uint4*)to = pack8<DT>(y);
    *(uint4*)(to + second) = pack8<DT>(y + 8);
  }
}

}  // namespace vib3

using namespace vib3;

extern "C" int vib3_launch_mla_append(const vib3_mla_append* args, void* stream) {
  if (!args) return VIB3_ERR_BAD_POINTER;
  const vib3_mla_append& a = *args;
  if (const int rc = check_cache(a.cache)) return rc;
  if (a.kv_dtype != VIB3_DT_F32 && !mla_dtype(a.kv_dtype)) return VIB3_ERR_UNSUPPORTED;
  if (a.tokens < 0 || (a.q_rope && (a.heads < 1 || a.heads > 65535))) return VIB3_ERR_BAD_COUNT;
  if (a.tokens == 0) return 0;
  if (!a.seqs || !a.positions || !a.inv_freq || !mla_aligned(a.kv) || !mla_stride(a.kv_stride))
    return VIB3_ERR_BAD_POINTER;
  if (a.norm_weight && !mla_aligned(a.norm_weight)) return VIB3_ERR_BAD_POINTER;
  if (a.kv_out && (!mla_aligned(a.kv_out) || !mla_stride(a.kv_out_stride))) return VIB3_ERR_BAD_POINTER;
  const int kv_blocks = (a.tokens + 3) / 4;
  if (a.q_rope) {
    if (!mla_aligned(a.q_rope) || !mla_aligned(a.q_out) || !mla_stride(a.q_token_stride) || !mla_stride(a.q_head_stride) ||
        !mla_stride(a.q_out_token_stride) || !mla_stride(a.q_out_head_stride))
      return VIB3_ERR_BAD_POINTER;
  }
  const int64_t blocks = kv_blocks + (a.q_rope ? (int64_t)a.tokens : 0);
  if (blocks > 0x7fffffff) return VIB3_ERR_BAD_COUNT;
  auto kernel = a.cache.dtype == VIB3_DT_F16 ? k_mla_append<VIB3_DT_F16> : k_mla_append<VIB3_DT_BF16>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, a, kv_blocks);
  VIB3_RETURN_LAUNCH();
}
