// gqa_chunk.hip — causal attention of each sequence's newest tokens over the paged key/value cache.
#include "gqa_simple.h"

namespace vib3 {
namespace {

template <int DT, int D>
__global__ __launch_bounds__(256) void k_gqa_chunk(vib3_gqa_chunk a) {
  const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (w >= (int64_t)a.q_tokens * a.heads) return;
  const int t = (int)(w / a.heads), h = (int)(w % a.heads);
  for (int s = 0; s < a.cache.num_seqs; s++) {
    const int q0 = min(max(a.cu_q[s], 0), a.q_tokens), q1 = min(a.cu_q[s + 1], a.q_tokens);
    if (t < q0 || t >= q1) continue;
    attend_simple<DT, D>(a.cache, s, gqa_len(a.cache, a.lens[s]) - (q1 - t), h / (a.heads / a.cache.kv_heads),
                         (const uint16_t*)a.q + t * a.q_token_stride + h * a.q_head_stride, a.scale, a.window, a.sinks,
                         (uint16_t*)a.out + t * a.out_token_stride + h * a.out_head_stride);
    return;
  }
}

template <int DT>
void launch_chunk(const vib3_gqa_chunk& a, hipStream_t st) {
  auto kernel = a.cache.dim == 64 ? k_gqa_chunk<DT, 64> : a.cache.dim == 128 ? k_gqa_chunk<DT, 128> : k_gqa_chunk<DT, 256>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)(((int64_t)a.q_tokens * a.heads + 3) / 4)), dim3(256), 0, st, a);
}

}  // namespace
}  // namespace vib3

using namespace vib3;

extern "C" size_t vib3_gqa_chunk_workspace_bytes(const vib3_gqa_chunk* args) {
  if (!args || check_gqa_cache(args->cache) || args->q_tokens < 0 || !gqa_heads(args->heads, args->cache.kv_heads)) return 0;
  return 256;
}

extern "C" int vib3_launch_gqa_chunk(const vib3_gqa_chunk* args, void* stream) {
  if (!args) return VIB3_ERR_BAD_POINTER;
  const vib3_gqa_chunk& a = *args;
  if (const int rc = check_gqa_cache(a.cache)) return rc;
  if (!__builtin_isfinite(a.scale)) return VIB3_ERR_UNSUPPORTED;
  if (!gqa_heads(a.heads, a.cache.kv_heads) || a.q_tokens < 0 || a.window < 0 || a.sinks < 0) return VIB3_ERR_BAD_COUNT;
  if ((int64_t)a.q_tokens * a.heads > 0x7fffffff) return VIB3_ERR_BAD_COUNT;
  if (a.q_tokens == 0 || a.cache.num_seqs == 0) return 0;
  if (!a.cu_q || !a.lens || !mla_aligned(a.q) || !mla_aligned(a.out) || !mla_stride(a.q_token_stride) || !mla_stride(a.q_head_stride) ||
      !mla_stride(a.out_token_stride) || !mla_stride(a.out_head_stride) || !a.workspace || ((uintptr_t)a.workspace & 255))
    return VIB3_ERR_BAD_POINTER;
  if (a.workspace_bytes < vib3_gqa_chunk_workspace_bytes(&a)) return VIB3_ERR_WORKSPACE;
  if (a.cache.dtype == VIB3_DT_F16) launch_chunk<VIB3_DT_F16>(a, (hipStream_t)stream);
  else launch_chunk<VIB3_DT_BF16>(a, (hipStream_t)stream);
  VIB3_RETURN_LAUNCH();
}
