// gqa_append.hip — new tokens into the paged key/value cache: RMSNorm of each head's query and key and their rotation, in one launch.
//
// A workgroup takes one token: its rows are the heads of q, k and v, one after the other, and D / 16 lanes share a row, 16 elements
// each, which are 8 pairs of the rotation. The cosines and sines are formed once a token (the angle and its reduction in 64 bits:
// positions reach 10^6 radians, where f32 angles are off by 0.03) while the first rows are on their way; a row's successor is loaded before
// the row is stored.
//
// Bound by HBM for prompts (6007 tokens of 40 + 8 + 8 heads of 128 from f32: 258 MB in 57 us, 4.5 TB/s; a copy of 2 GB 5.0), by the launch and
// its chain of reads (sequence, page number, row) for single tokens (5 us).
#include "gqa.h"
#include "scan.h"

namespace vib3 {
namespace {

template <int DT, int D>
__global__ __launch_bounds__(256) void k_gqa_append(vib3_gqa_append a) {
  constexpr int kLanes = D / 16;  // of a row
  __shared__ float2 turns[D / 2];
  const int tid = (int)threadIdx.x, t = (int)wide_block();
  if ((unsigned)t >= (unsigned)a.tokens) return;
  const int s = a.seqs[t], p = a.positions[t];
  if ((unsigned)s >= (unsigned)a.cache.num_seqs || p < 0) return;
  const int64_t cached = gqa_token(a.cache, s, p);
  const int half = a.rot / 2, kv = a.cache.kv_heads, qh = a.q ? a.heads : 0;
  const int u = tid % kLanes;
  // this lane's two runs of eight elements of a row that is turned
  const bool turned = u * 16 < a.rot;
  const int first = turned && !a.interleaved ? 8 * u : 16 * u, second = turned && !a.interleaved ? first + half : first + 8;
  const int rows = qh + (cached >= 0 ? 2 * kv : 0);
  float x[16];
  auto fetch = [&](int row) {
    const int g = row < qh ? row : row < qh + kv ? row - qh : row - qh - kv;
    const void* src = row < qh ? a.q : row < qh + kv ? a.k : a.v;
    const int64_t at = row < qh        ? (int64_t)t * a.q_token_stride + (int64_t)g * a.q_head_stride
                       : row < qh + kv ? (int64_t)t * a.k_token_stride + (int64_t)g * a.k_head_stride
                                       : (int64_t)t * a.v_token_stride + (int64_t)g * a.v_head_stride;
    load8(src, a.src_dtype, at + first, x);
    load8(src, a.src_dtype, at + second, x + 8);
  };
  int row = tid / kLanes;
  if (row < rows) fetch(row);
  if (tid < half) {
    double angle = (double)p * (double)a.inv_freq[tid] * 0.15915494309189535;  // in turns
    angle -= __builtin_rint(angle);
    float sn, cs;
    sincospif(2.0f * (float)angle, &sn, &cs);
    turns[tid] = make_float2(a.rope_scale * cs, a.rope_scale * sn);
  }
  __syncthreads();
  for (; row < rows; row += 256 / kLanes) {
    const bool is_value = row >= qh + kv;
    const void* norm = row < qh ? a.q_norm : is_value ? nullptr : a.k_norm;
    float y[16];
    if (norm) {
      float w[16], ss = 0.0f;
      load8(norm, a.norm_dtype, first, w);
      load8(norm, a.norm_dtype, second, w + 8);
#pragma unroll
      for (int i = 0; i < 16; i++) ss = __builtin_fmaf(x[i], x[i], ss);
#pragma unroll
      for (int d = 1; d < kLanes; d *= 2) ss += __shfl_xor(ss, d);
      const float inv = 1.0f / sqrtf(ss / (float)D + a.norm_eps);
#pragma unroll
      for (int i = 0; i < 16; i++) y[i] = x[i] * inv * w[i];
    } else {
#pragma unroll
      for (int i = 0; i < 16; i++) y[i] = x[i];
    }
    if (turned && !is_value) {
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const float2 c = turns[8 * u + i];
        const float y0 = a.interleaved ? y[2 * i] : y[i], y1 = a.interleaved ? y[2 * i + 1] : y[i + 8];
        const float z0 = y0 * c.x - y1 * c.y, z1 = y0 * c.y + y1 * c.x;
        if (a.interleaved) y[2 * i] = z0, y[2 * i + 1] = z1;
        else y[i] = z0, y[i + 8] = z1;
      }
    }
    uint16_t* to;
    if (row < qh) to = (uint16_t*)a.q_out + (int64_t)t * a.q_out_token_stride + (int64_t)row * a.q_out_head_stride;
    else if (!is_value) to = (uint16_t*)a.cache.keys + cached + (int64_t)(row - qh) * a.cache.head_stride;
    else to = (uint16_t*)a.cache.values + cached + (int64_t)(row - qh - kv) * a.cache.head_stride;
    if (row + 256 / kLanes < rows) fetch(row + 256 / kLanes);
    *(uint4*)(to + first) = pack8<DT>(y);
    *(uint4*)(to + second) = pack8<DT>(y + 8);
  }
}

template <int DT>
void launch_append(const vib3_gqa_append& a, hipStream_t st) {
  auto kernel = a.cache.dim == 64 ? k_gqa_append<DT, 64> : a.cache.dim == 128 ? k_gqa_append<DT, 128> : k_gqa_append<DT, 256>;
  hipLaunchKernelGGL(kernel, wide_grid(a.tokens), dim3(256), 0, st, a);
}

}  // namespace
}  // namespace vib3

using namespace vib3;

extern "C" int vib3_launch_gqa_append(const vib3_gqa_append* args, void* stream) {
  if (!args) return VIB3_ERR_BAD_POINTER;
  const vib3_gqa_append& a = *args;
  if (const int rc = check_gqa_cache(a.cache)) return rc;
  const auto float_dtype = [](int dt) { return dt == VIB3_DT_F32 || mla_dtype(dt); };
  if (!float_dtype(a.src_dtype) || ((a.q_norm || a.k_norm) && !float_dtype(a.norm_dtype)) || a.rot % 16 || a.rot < 0 ||
      a.rot > a.cache.dim)
    return VIB3_ERR_UNSUPPORTED;
  if (a.tokens < 0 || (a.q && !gqa_heads(a.heads, a.cache.kv_heads))) return VIB3_ERR_BAD_COUNT;
  if (a.tokens == 0) return 0;
  if (!a.seqs || !a.positions || (a.rot && !a.inv_freq) || !mla_aligned(a.k) || !mla_aligned(a.v) || !mla_stride(a.k_token_stride) ||
      !mla_stride(a.k_head_stride) || !mla_stride(a.v_token_stride) || !mla_stride(a.v_head_stride))
    return VIB3_ERR_BAD_POINTER;
  if ((a.q_norm && !mla_aligned(a.q_norm)) || (a.k_norm && !mla_aligned(a.k_norm))) return VIB3_ERR_BAD_POINTER;
  if (a.q && (!mla_aligned(a.q) || !mla_aligned(a.q_out) || !mla_stride(a.q_token_stride) || !mla_stride(a.q_head_stride) ||
              !mla_stride(a.q_out_token_stride) || !mla_stride(a.q_out_head_stride)))
    return VIB3_ERR_BAD_POINTER;
  if (a.cache.dtype == VIB3_DT_F16) launch_append<VIB3_DT_F16>(a, (hipStream_t)stream);
  else launch_append<VIB3_DT_BF16>(a, (hipStream_t)stream);
  VIB3_RETURN_LAUNCH();
}
