// gqa_decode.hip — attention of single query tokens over the paged key/value cache.
#include "gqa_simple.h"

namespace vib3 {

constexpr int kGqaMaxRows = 65536;

template <int DT, int D>
__global__ __launch_bounds__(256) void k_gqa_decode(vib3_gqa_decode a) {
  const int w = (int)(blockIdx.x * 4 + (threadIdx.x >> 6));
  if (w >= a.rows * a.heads) return;
  const int r = w / a.heads, h = w % a.heads;
  const int s = a.seqs ? a.seqs[r] : r;
  const int len = (unsigned)s < (unsigned)a.cache.num_seqs ? gqa_len(a.cache, a.lens[r]) : 0;
  attend_simple<DT, D>(a.cache, s, len - 1, h / (a.heads / a.cache.kv_heads),
                       (const uint16_t*)a.q + r * a.q_row_stride + h * a.q_head_stride, a.scale, a.window, a.sinks,
                       (uint16_t*)a.out + r * a.out_row_stride + h * a.out_head_stride);
}

template <int DT>
void launch_decode(const vib3_gqa_decode& a, hipStream_t st) {
  auto kernel = a.cache.dim == 64 ? k_gqa_decode<DT, 64> : a.cache.dim == 128 ? k_gqa_decode<DT, 128> : k_gqa_decode<DT, 256>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)((a.rows * a.heads + 3) / 4)), dim3(256), 0, st, a);
}

}  // namespace vib3

using namespace vib3;

extern "C" size_t vib3_gqa_decode_workspace_bytes(const vib3_gqa_decode* args) {
  if (!args || check_gqa_cache(args->cache) || args->rows < 0 || args->rows > kGqaMaxRows ||
      !gqa_heads(args->heads, args->cache.kv_heads))
    return 0;
  return 256;
}

extern "C" int vib3_launch_gqa_decode(const vib3_gqa_decode* args, void* stream) {
  if (!args) return VIB3_ERR_BAD_POINTER;
  const vib3_gqa_decode& a = *args;
  if (const int rc = check_gqa_cache(a.cache)) return rc;
  if (!__builtin_isfinite(a.scale)) return VIB3_ERR_UNSUPPORTED;
  if (a.rows < 0 || a.rows > kGqaMaxRows || !gqa_heads(a.heads, a.cache.kv_heads) || a.window < 0 || a.sinks < 0)
    return VIB3_ERR_BAD_COUNT;
  if (a.rows == 0) return 0;
  if (!a.lens || !mla_aligned(a.q) || !mla_aligned(a.out) || !mla_stride(a.q_row_stride) || !mla_stride(a.q_head_stride) ||
      !mla_stride(a.out_row_stride) || !mla_stride(a.out_head_stride) || !a.workspace || ((uintptr_t)a.workspace & 255))
    return VIB3_ERR_BAD_POINTER;
  if (a.workspace_bytes < vib3_gqa_decode_workspace_bytes(&a)) return VIB3_ERR_WORKSPACE;
  if (a.cache.dtype == VIB3_DT_F16) launch_decode<VIB3_DT_F16>(a, (hipStream_t)stream);
  else launch_decode<VIB3_DT_BF16>(a, (hipStream_t)stream);
  VIB3_RETURN_LAUNCH();
}
