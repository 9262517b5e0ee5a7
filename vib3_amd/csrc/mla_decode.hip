// mla_decode.hip — attention of single query tokens over the paged latent cache, absorbed form.
#include "mla.h"

namespace vib3 {

constexpr int kMlaMaxRows = 65536;

// One workgroup per (row, head). The query goes into the latent space (thread c holds column c),
// each wave then takes every fourth cached token with a softmax of its own (running maximum and
// sum; lane l holds eight latent elements), the four waves are joined, and the weighted latent
// goes through W_uv, a wave per output element.
template <int DT>
__global__ __launch_bounds__(256) void k_mla_decode(vib3_mla_decode a) {
  const int r = (int)blockIdx.x, h = (int)blockIdx.y, tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int rank = a.cache.rank, rope = a.cache.rope;
  __shared__ float q[512 + 64];
  __shared__ float acc[4][512];
  __shared__ float stat[4][2];
  const uint16_t* qn = (const uint16_t*)a.q_nope + (int64_t)r * a.q_nope_row_stride + (int64_t)h * a.q_nope_head_stride;
  const uint16_t* qr = (const uint16_t*)a.q_rope + (int64_t)r * a.q_rope_row_stride + (int64_t)h * a.q_rope_head_stride;
  const uint16_t* w = (const uint16_t*)a.kv_b + (size_t)h * (a.nope + a.v_dim) * rank;
  for (int c = tid; c < rank; c += 256) {
    float s = 0.0f;
    if (a.kv_b) {
      for (int n = 0; n < a.nope; n++) s = __builtin_fmaf(to_f32<DT>(qn[n]), to_f32<DT>(w[(size_t)n * rank + c]), s);
    } else {
      s = to_f32<DT>(qn[c]);
    }
    q[c] = s;
  }
  if (tid < rope) q[rank + tid] = to_f32<DT>(qr[tid]);
  __syncthreads();
  const int seq = a.seqs ? a.seqs[r] : r;
  const int len = (unsigned)seq < (unsigned)a.cache.num_seqs ? clamp_len(a.cache, a.lens[r]) : 0;
  const bool mine = lane * 8 < rank;
  float m = -__builtin_huge_valf(), l = 0.0f, o[8] = {};
  for (int j = wave; j < len; j += 4) {
    const uint16_t* row = cache_row(a.cache, seq, j);
    if (!row) continue;
    float c[8], s = 0.0f;
    if (mine) {
      unpack8<DT>(*(const uint4*)(row + lane * 8), c);
      for (int i = 0; i < 8; i++) s = __builtin_fmaf(c[i], q[lane * 8 + i], s);
    }
    if (lane < rope) s = __builtin_fmaf(to_f32<DT>(row[rank + lane]), q[rank + lane], s);
    s = wave_sum(s) * a.scale;
    const float mn = fmaxf(m, s), base = mn == -__builtin_huge_valf() ? 0.0f : mn;
    const float f = expf(m - base), p = expf(s - base);
    l = l * f + p;
    if (mine)
      for (int i = 0; i < 8; i++) o[i] = o[i] * f + p * c[i];
    m = mn;
  }
  if (mine)
    for (int i = 0; i < 8; i++) acc[wave][lane * 8 + i] = o[i];
  if (lane == 0) {
    stat[wave][0] = m;
    stat[wave][1] = l;
  }
  __syncthreads();
  float mm = fmaxf(fmaxf(stat[0][0], stat[1][0]), fmaxf(stat[2][0], stat[3][0]));
  if (mm == -__builtin_huge_valf()) mm = 0.0f;
  float f[4], sum = 0.0f;
  for (int i = 0; i < 4; i++) {
    f[i] = expf(stat[i][0] - mm);
    sum += f[i] * stat[i][1];
  }
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  for (int c = tid; c < rank; c += 256)
    q[c] = (f[0] * acc[0][c] + f[1] * acc[1][c] + f[2] * acc[2][c] + f[3] * acc[3][c]) * inv;
  __syncthreads();
  uint16_t* out = (uint16_t*)a.out + (int64_t)r * a.out_row_stride + (int64_t)h * a.out_head_stride;
  if (!a.kv_b) {
    for (int c = tid; c < rank; c += 256) out[c] = from_f32<DT>(q[c]);
    return;
  }
  for (int v = wave; v < a.v_dim; v += 4) {
    float s = 0.0f;
    if (mine) {
      float x[8];
      unpack8<DT>(*(const uint4*)(w + (size_t)(a.nope + v) * rank + lane * 8), x);
      for (int i = 0; i < 8; i++) s = __builtin_fmaf(x[i], q[lane * 8 + i], s);
    }
    s = wave_sum(s);
    if (lane == 0) out[v] = from_f32<DT>(s);
  }
}

}  // namespace vib3

using namespace vib3;

extern "C" size_t vib3_mla_decode_workspace_bytes(const vib3_mla_decode* args) {
  if (!args || args->rows < 0 || args->rows > kMlaMaxRows || args->heads < 1 || args->heads > 128) return 0;
  return 256;
}

extern "C" int vib3_launch_mla_decode(const vib3_mla_decode* args, void* stream) {
  if (!args) return VIB3_ERR_BAD_POINTER;
  const vib3_mla_decode& a = *args;
  if (const int rc = check_cache(a.cache)) return rc;
  if (a.rows < 0 || a.rows > kMlaMaxRows || a.heads < 1 || a.heads > 128) return VIB3_ERR_BAD_COUNT;
  if (a.kv_b && (a.nope < 32 || a.nope > 256 || a.nope % 32 || a.v_dim < 32 || a.v_dim > 256 || a.v_dim % 32))
    return VIB3_ERR_UNSUPPORTED;
  if (a.rows == 0) return 0;
  if (!a.lens || !mla_aligned(a.q_nope) || !mla_aligned(a.q_rope) || !mla_aligned(a.out) ||
      (a.kv_b && !mla_aligned(a.kv_b)) || !mla_stride(a.q_nope_row_stride) || !mla_stride(a.q_nope_head_stride) ||
      !mla_stride(a.q_rope_row_stride) || !mla_stride(a.q_rope_head_stride) || !mla_stride(a.out_row_stride) ||
      !mla_stride(a.out_head_stride) || !a.workspace || ((uintptr_t)a.workspace & 255))
    return VIB3_ERR_BAD_POINTER;
  if (a.workspace_bytes < vib3_mla_decode_workspace_bytes(args)) return VIB3_ERR_WORKSPACE;
  auto kernel = a.cache.dtype == VIB3_DT_F16 ? k_mla_decode<VIB3_DT_F16> : k_mla_decode<VIB3_DT_BF16>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)a.rows, (unsigned)a.heads), dim3(256), 0, (hipStream_t)stream, a);
  VIB3_RETURN_LAUNCH();
}
