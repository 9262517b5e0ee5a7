// mla_prefill.hip — causal attention of whole prompts, expanded form (a key and a value per head).
#include "mla.h"

namespace vib3 {

// A wave per (query, head): running maximum and sum over the visible keys, one key at a time.
template <int DT>
__global__ __launch_bounds__(256) void k_mla_prefill(vib3_mla_prefill a) {
  const int i = (int)blockIdx.x * 4 + ((int)threadIdx.x >> 6), h = (int)blockIdx.y, lane = lane_id();
  if (i >= a.q_tokens) return;
  int s = 0;  // the sequence of query i
  while (s < a.num_seqs && min(a.cu_q[s + 1], a.q_tokens) <= i) s++;
  if (s == a.num_seqs || i < a.cu_q[s]) return;
  const int q0 = max(a.cu_q[s], 0), q1 = min(a.cu_q[s + 1], a.q_tokens);
  const int k0 = min(max(a.cu_k[s], 0), a.k_tokens), k1 = min(max(a.cu_k[s + 1], k0), a.k_tokens);
  const int end = min(k1, k0 + i - q0 + (k1 - k0) - (q1 - q0) + 1);
  const uint16_t* qn = (const uint16_t*)a.q_nope + (int64_t)i * a.q_nope_token_stride + (int64_t)h * a.q_nope_head_stride;
  const uint16_t* qr = (const uint16_t*)a.q_rope + (int64_t)i * a.q_rope_token_stride + (int64_t)h * a.q_rope_head_stride;
  const bool n2 = a.nope > 64, v2 = a.v_dim > 64;
  const float qa = to_f32<DT>(qn[lane]), qb = n2 ? to_f32<DT>(qn[64 + lane]) : 0.0f;
  const float qc = lane < a.rope ? to_f32<DT>(qr[lane]) : 0.0f;
  float m = -__builtin_huge_valf(), l = 0.0f, oa = 0.0f, ob = 0.0f;
  for (int j = k0; j < end; j++) {
    const uint16_t* kv = (const uint16_t*)a.kv + (int64_t)j * a.kv_token_stride + (int64_t)h * a.kv_head_stride;
    float x = qa * to_f32<DT>(kv[lane]);
    if (n2) x = __builtin_fmaf(qb, to_f32<DT>(kv[64 + lane]), x);
    if (lane < a.rope) x = __builtin_fmaf(qc, to_f32<DT>(((const uint16_t*)a.k_rope)[(int64_t)j * a.k_rope_stride + lane]), x);
    x = wave_sum(x) * a.scale;
    const float mn = fmaxf(m, x), base = mn == -__builtin_huge_valf() ? 0.0f : mn;
    const float f = expf(m - base), p = expf(x - base);
    l = l * f + p;
    oa = oa * f + p * to_f32<DT>(kv[a.nope + lane]);
    if (v2) ob = ob * f + p * to_f32<DT>(kv[a.nope + 64 + lane]);
    m = mn;
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  uint16_t* out = (uint16_t*)a.out + (int64_t)i * a.out_token_stride + (int64_t)h * a.out_head_stride;
  out[lane] = from_f32<DT>(oa * inv);
  if (v2) out[64 + lane] = from_f32<DT>(ob * inv);
}

}  // namespace vib3

using namespace vib3;

extern "C" int vib3_launch_mla_prefill(const vib3_mla_prefill* args, void* stream) {
  if (!args) return VIB3_ERR_BAD_POINTER;
  const vib3_mla_prefill& a = *args;
  if (!mla_dtype(a.dtype) || (a.nope != 64 && a.nope != 128) || (a.v_dim != 64 && a.v_dim != 128) ||
      (a.rope != 32 && a.rope != 64))
    return VIB3_ERR_UNSUPPORTED;
  if (a.heads < 1 || a.heads > 65535 || a.num_seqs < 0 || a.q_tokens < 0 || a.k_tokens < 0 ||
      ((int64_t)a.q_tokens + 3) / 4 * a.heads > 0x7fffffff)
    return VIB3_ERR_BAD_COUNT;
  if (a.q_tokens == 0 || a.num_seqs == 0) return 0;
  if (!a.cu_q || !a.cu_k || !mla_aligned(a.q_nope) || !mla_aligned(a.q_rope) || !mla_aligned(a.out) ||
      (a.k_tokens && (!mla_aligned(a.kv) || !mla_aligned(a.k_rope))) || !mla_stride(a.q_nope_token_stride) ||
      !mla_stride(a.q_nope_head_stride) || !mla_stride(a.q_rope_token_stride) || !mla_stride(a.q_rope_head_stride) ||
      !mla_stride(a.kv_token_stride) || !mla_stride(a.kv_head_stride) || !mla_stride(a.k_rope_stride) ||
      !mla_stride(a.out_token_stride) || !mla_stride(a.out_head_stride))
    return VIB3_ERR_BAD_POINTER;
  auto kernel = a.dtype == VIB3_DT_F16 ? k_mla_prefill<VIB3_DT_F16> : k_mla_prefill<VIB3_DT_BF16>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)((a.q_tokens + 3) / 4), (unsigned)a.heads), dim3(256), 0, (hipStream_t)stream, a);
  VIB3_RETURN_LAUNCH();
}
