// mla_prefill.hip — causal attention of whole prompts, expanded form (a key and a value per head).
//
// Bound by the matrix cores: 2 (nope + rope + v_dim) flops per visible (query, key, head), 640 at 128 + 64 + 128, against
// bytes that are read once per 256 queries. 12288 tokens of 64 heads (3.09 TFLOP, bf16): 3.0 to 3.2 ms, 0.97 to 1.03 PFLOP/s, where a
// large library product reaches 1.22; shorter prompts end unevenly (a workgroup a CU). The reads from LDS, 32 queries a wave,
// take as long as the products, 2600 cycles a tile of eight waves. A workgroup takes 32 queries of one head per wave and walks over
// the keys, 64 at a time, with a running maximum and sum per query.
//
// Scores are formed transposed, S^T = K . Q^T, so that a lane holds one query's scores of 32 of the 64 keys (the other lane
// of the pair l, l + 32 the rest): the maximum and sum are almost all within a lane, and the probabilities, packed in pairs of
// 16 bits, are as they stand the B operand of O^T = V^T . P^T (the keys' order along k is free as long as V^T is read in the
// same one, which the transposing LDS reads allow). The scores of the next 64 keys are formed next to the softmax of these, so that the
// matrix cores and the vector units have work of one wave at a time. (The two waves of a SIMD in turns, one at its products
// while the other is at its softmax, with a barrier after each: 3.4 to 3.6 ms.)
//
// Keys and values go straight from memory to LDS, double-buffered, the shared rotary key once per workgroup and tile.
// 16-byte chunk c of an LDS row lies at c ^ a function of the row, which spreads the reads over the banks.
#include <type_traits>

#include "mla.h"

namespace vib3 {

constexpr int kKeys = 64;  // keys of one step

// What rows behind the last key are read from.
__device__ const uint4 zero_key[128 / 8] = {};

// Operand layouts of the 32x32x16 products: lane l holds row (A) or column (B) l % 32 at k = 8 (l / 32) + 0..7; of the result,
// column l % 32, element i in row 8 (i / 4) + 4 (l / 32) + i % 4.
typedef float f32x16 __attribute__((ext_vector_type(16)));

template <int DT>
__device__ __forceinline__ f32x16 mma_wide(s16x8 a, s16x8 b, f32x16 c) {
  if (DT == VIB3_DT_F16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// Where chunk 0 of a row lies, for rows of C chunks: 16 (or 8) rows in a row-wise read of one chunk fall into different banks.
template <int C>
__device__ __forceinline__ int key_swizzle(int row) {
  return C == 16 ? row & 15 : C == 8 ? (row >> 1) & 7 : (row >> 2) & 3;
}

// The same for values, of which a transposing read takes 64 bytes of each of 8 rows.
template <int C>
__device__ __forceinline__ int value_swizzle(int row) {
  return C == 16 ? (row & 3) << 2 : ((row >> 1) & 1) << 2;
}

// Maximum and sum over the lanes l and l + 32.
__device__ __forceinline__ float pair_max(float v) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float pair_sum(float v) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

// A word's two 16-bit elements with zeros in the place of infinities and NaN.
template <int DT>
__device__ __forceinline__ uint32_t finite_only(uint32_t w) {
  constexpr uint32_t e = DT == VIB3_DT_F16 ? 0x7c00u : 0x7f80u;
  return ((w & e) == e ? 0u : w & 0xffffu) | ((w & (e << 16)) == (e << 16) ? 0u : w & 0xffff0000u);
}

// The queries of a workgroup: sequence, first query in it, and its queries and keys.
struct Block {
  int q0, nq, k0, nk, first;
};

// Blocks of `size` queries of all sequences are numbered in order, a sequence's last block first (it sees the most keys). Each wave
// finds block b by itself, 64 sequences at a time; false: there is no block b.
__device__ bool find_block(const vib3_mla_prefill& a, int b, int size, Block* out) {
  const int lane = lane_id();
  for (int s0 = 0; s0 < a.num_seqs; s0 += 64) {
    const int s = s0 + lane;
    int q0 = 0, n = 0;
    if (s < a.num_seqs) {
      q0 = min(max(a.cu_q[s], 0), a.q_tokens);
      n = max(min(a.cu_q[s + 1], a.q_tokens) - q0, 0);
    }
    const int blocks = (n + size - 1) / size;
    int upto = blocks;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int v = __shfl_up(upto, d);
      if (lane >= d) upto += v;
    }
    const uint64_t hit = __ballot(b < upto);
    if (hit) {
      const int l = __ffsll((unsigned long long)hit) - 1;
      const int last = __builtin_amdgcn_readlane(upto, l);
      out->q0 = __builtin_amdgcn_readlane(q0, l);
      out->nq = __builtin_amdgcn_readlane(n, l);
      out->first = (last - 1 - b) * size;
      const int q = s0 + l;
      const int k0 = min(max(a.cu_k[q], 0), a.k_tokens);
      out->k0 = k0;
      out->nk = max(min(a.cu_k[q + 1], a.k_tokens) - k0, 0);
      return true;
    }
    b -= __builtin_amdgcn_readlane(upto, 63);
  }
  return false;
}

template <int DT, int N, int P, int V, int WAVES>
__global__ __launch_bounds__(WAVES * 64, WAVES / 4) void k_mla_prefill(vib3_mla_prefill a) {
  constexpr int NC = N / 8, PC = P / 8, VC = V / 8;    // 16-byte chunks of a row
  constexpr int KS = (N + P) / 16;                     // k steps of the scores
  constexpr int VB = V / 32;                           // 32-column blocks of the sums
  constexpr int kSize = WAVES * 32;                    // queries of a workgroup
  __shared__ __align__(1024) uint8_t ktile[2][kKeys * N * 2];
  __shared__ __align__(1024) uint8_t rtile[2][kKeys * P * 2];
  __shared__ __align__(1024) uint8_t vtile[2][kKeys * V * 2];
  __shared__ int odd_values[2][WAVES];                 // whether a wave's part of a tile's values held infinities or NaN

  const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int half = lane >> 5, col = lane & 31;
  const int h = (int)(blockIdx.x % (unsigned)a.heads);
  Block bl;
  if (!find_block(a, (int)(blockIdx.x / (unsigned)a.heads), kSize, &bl)) return;

  // this lane's query (in its sequence) and the last key it sees (-1: none)
  const int qi = bl.first + wave * 32 + col;
  const int shift = bl.nk - bl.nq;
  const int limit = qi < bl.nq ? max(qi + shift, -1) : -1;
  const int w_first = bl.first + wave * 32;                            // the wave's first query
  const int low = w_first + 31 < bl.nq ? w_first + shift : -1;         // every query of the wave sees keys up to here
  const int high = min(w_first + 31, bl.nq - 1) + shift;               // no query sees more (if it has any)
  const int my_tiles = w_first < bl.nq && high >= 0 ? high / kKeys + 1 : 0;
  const int top_key = min(bl.first + kSize, bl.nq) - 1 + shift;
  const int tiles = top_key >= 0 ? top_key / kKeys + 1 : 0;            // of the workgroup
  const int first_masked = max(bl.first + shift + 1, 0) / kKeys;       // from here on some query does not see all of a tile

  // queries: the B operand, this lane's query at k = 16 s + 8 half
  const float scale = exponent_scale(a.scale);
  const uint32_t flip = sign_flip(a.scale);
  s16x8 q[KS];
  {
    const int64_t t = bl.q0 + min(qi, bl.nq - 1);
    const uint16_t* qn = (const uint16_t*)a.q_nope + t * a.q_nope_token_stride + (int64_t)h * a.q_nope_head_stride;
    const uint16_t* qr = (const uint16_t*)a.q_rope + t * a.q_rope_token_stride + (int64_t)h * a.q_rope_head_stride;
#pragma unroll
    for (int s = 0; s < KS; s++) {
      uint4 v = *(const uint4*)(s < N / 16 ? qn + 16 * s + 8 * half : qr + 16 * (s - N / 16) + 8 * half);
      v.x ^= flip; v.y ^= flip; v.z ^= flip; v.w ^= flip;
      q[s] = __builtin_bit_cast(s16x8, v);
    }
  }
  VIB3_WAIT_VM(0);  // here, once: a wait inside the loop would drain the tiles' loads

  // Loads: a wave takes every WAVES-th run of 64 chunks of each part of a tile; its first row in it and the lane's place.
  const uint16_t* kv = (const uint16_t*)a.kv + (int64_t)bl.k0 * a.kv_token_stride + (int64_t)h * a.kv_head_stride;
  const uint16_t* kr = (const uint16_t*)a.k_rope + (int64_t)bl.k0 * a.k_rope_stride;
  auto load_part = [&](auto chunks, const uint16_t* src, int64_t stride, int tile, uint8_t* dst, auto swizzle) {
    constexpr int C = decltype(chunks)::value, kRows = 64 / C, kRuns = kKeys / kRows;
#pragma unroll
    for (int i = 0; i < (kRuns + WAVES - 1) / WAVES; i++) {
      const int run = i * WAVES + wave;
      if (kRuns % WAVES && run >= kRuns) break;
      const int row = run * kRows + lane / C;
      const int j = tile * kKeys + row;
      const uint16_t* p = src + (int64_t)j * stride;
      const uint8_t* at = (const uint8_t*)(j < bl.nk ? p : (const uint16_t*)zero_key);
      load_to_lds16(at + ((lane % C) ^ swizzle(row)) * 16, (lds_u8*)dst + run * 1024);
    }
  };
  auto load_keys = [&](int tile) {
    load_part(std::integral_constant<int, NC>{}, kv, a.kv_token_stride, tile, ktile[tile & 1], [](int r) { return key_swizzle<NC>(r); });
    load_part(std::integral_constant<int, PC>{}, kr, a.k_rope_stride, tile, rtile[tile & 1], [](int r) { return key_swizzle<PC>(r); });
  };
  auto load_values = [&](int tile) {
    load_part(std::integral_constant<int, VC>{}, kv + N, a.kv_token_stride, tile, vtile[tile & 1], [](int r) { return value_swizzle<VC>(r); });
  };
  // A masked place has probability 0, and 0 times an infinity or a NaN is NaN: in tiles with masked places the values that
  // this wave has loaded are cleared of those, and whether there were any is noted.
  auto clear_values = [&](int tile) {
    bool odd = false;
    constexpr int kRuns = kKeys * VC / 64;
#pragma unroll
    for (int i = 0; i < (kRuns + WAVES - 1) / WAVES; i++) {
      const int run = i * WAVES + wave;
      if (kRuns % WAVES && run >= kRuns) break;
      uint4* at = (uint4*)(vtile[tile & 1] + run * 1024 + lane * 16);
      const uint4 v = *at, w = make_uint4(finite_only<DT>(v.x), finite_only<DT>(v.y), finite_only<DT>(v.z), finite_only<DT>(v.w));
      if (v.x != w.x || v.y != w.y || v.z != w.z || v.w != w.w) {
        *at = w;
        odd = true;
      }
    }
    const int any = __any(odd);
    if (lane == 0) odd_values[tile & 1][wave] = any;
  };

  // S^T of a tile: two blocks of 32 keys
  auto form_scores = [&](int tile, f32x16* s) {
    const lds_u8* t = (lds_u8*)ktile[tile & 1] + col * N * 2;
    const lds_u8* u = (lds_u8*)rtile[tile & 1] + col * P * 2;
    const int k0 = fresh((half ^ key_swizzle<NC>(col)) * 16), u0 = fresh((half ^ key_swizzle<PC>(col)) * 16);
#pragma unroll
    for (int b = 0; b < 2; b++) s[b] = f32x16{};
#pragma unroll
    for (int k = 0; k < N / 16; k++)
#pragma unroll
      for (int b = 0; b < 2; b++) s[b] = mma_wide<DT>(lds_read16(t + b * 32 * N * 2 + (k0 ^ 32 * k)), q[k], s[b]);
#pragma unroll
    for (int k = 0; k < P / 16; k++)
#pragma unroll
      for (int b = 0; b < 2; b++)
        s[b] = mma_wide<DT>(lds_read16(u + b * 32 * P * 2 + (u0 ^ 32 * k)), q[N / 16 + k], s[b]);
  };

  f32x16 o[VB] = {};
  float m = -__builtin_huge_valf(), l = 0.0f;  // running maximum (of unscaled scores) and this lane's part of the sum
  f32x16 s[2];
  if (tiles > 0) {
    load_keys(0);
    wait_lds_loads();
    __syncthreads();
    load_keys(1);
    load_values(0);
    form_scores(0, s);
  }
  // this lane's place in a transposing read: row 4 half + (lane % 16) / 4, columns 16 ((lane / 16) % 2) + 4 (lane % 4)
  const int vrow = 4 * half + ((lane & 15) >> 2);
  const int vchunk = ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1);
  for (int n = 0; n < tiles; n++) {
    wait_lds_loads();
    const bool masked = n >= first_masked;
    if (masked) clear_values(n);
    __syncthreads();  // keys n + 1 and values n are in LDS; everyone is done with keys n and values n - 1
    if (n + 2 < tiles) load_keys(n + 2);
    if (n + 1 < tiles) load_values(n + 1);
    if (n >= my_tiles) continue;

    if (n * kKeys + kKeys - 1 > low) {
#pragma unroll
      for (int b = 0; b < 2; b++)
#pragma unroll
        for (int i = 0; i < 16; i++)
          if (n * kKeys + 32 * b + 8 * (i >> 2) + 4 * half + (i & 3) > limit) s[b][i] = -__builtin_huge_valf();
    }
    f32x16 s_next[2];
    form_scores(n + 1, s_next);  // past the last tile: of whatever lies there, and not used

    float top = s[0][0];
#pragma unroll
    for (int i = 1; i < 16; i++) top = fmaxf(top, s[0][i]);
#pragma unroll
    for (int i = 0; i < 16; i++) top = fmaxf(top, s[1][i]);
    top = pair_max(top);
    // The reference value of a query's exponentials follows its maximum only where that grew by more than kLag. (Each query by
    // itself: what others of the wave see does not change its result.)
    const bool grown = (top - m) * scale > kLag<DT> || (m == -__builtin_huge_valf() && top > m);
    if (__any(grown)) {
      const float f = grown ? __builtin_amdgcn_exp2f((m - top) * scale) : 1.0f;
      m = grown ? top : m;
      l *= f;
#pragma unroll
      for (int c = 0; c < VB; c++) o[c] *= f;
    }
    float base = m == -__builtin_huge_valf() ? 0.0f : m * scale;
    const bool far = __builtin_fabsf(base) > kFarExponent;
    if (__any(far)) {
      const float off = far ? m : 0.0f;
      base = far ? 0.0f : base;
#pragma unroll
      for (int b = 0; b < 2; b++)
#pragma unroll
        for (int i = 0; i < 16; i++) s[b][i] -= off;
    }
    base -= kProbShift<DT>;
    uint32_t p[16];
#pragma unroll
    for (int b = 0; b < 2; b++)
#pragma unroll
      for (int i = 0; i < 16; i += 2) {
        const float e0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][i], scale, -base));
        const float e1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][i + 1], scale, -base));
        l += e0 + e1;
        // Rounded for the matrix cores; the sum l takes them unrounded. (A remainder as a second summand takes a quarter to a third
        // more: 12288 tokens 3.06 -> 4.16 ms. Without it the result is off by 0.0019 to 0.0022 in bf16, a single rounding by 0.0016.)
        p[8 * b + (i >> 1)] = pack2<DT>(e0, e1);
      }
    lds_u8* const v = (lds_u8*)vtile[n & 1] + vrow * V * 2 + 8 * (lane & 1);
    const int v0 = fresh((vchunk ^ value_swizzle<VC>(vrow)) * 16);  // 16 and 8 rows further the swizzle is the same
    // V^T for 32 columns and 16 keys
    auto values = [&](int k, int c) {
      return join(lds_read_tr(v + 16 * k * V * 2 + (v0 ^ 64 * c)), lds_read_tr(v + (16 * k + 8) * V * 2 + (v0 ^ 64 * c)));
    };
    auto probs = [&](int k) { return __builtin_bit_cast(s16x8, make_uint4(p[4 * k], p[4 * k + 1], p[4 * k + 2], p[4 * k + 3])); };
#pragma unroll
    for (int k = 0; k < kKeys / 16; k++)
#pragma unroll
      for (int c = 0; c < VB; c++) o[c] = mma_wide<DT>(values(k, c), probs(k), o[c]);
    if (masked) {
      int odd = 0;
#pragma unroll
      for (int w = 0; w < WAVES; w++) odd |= odd_values[n & 1][w];
      if (__builtin_amdgcn_readfirstlane(odd)) {
        // What was cleared, for the queries that do see it: infinities times a probability of 0 are NaN, as in other tiles.
        // (Whether it is 0 is formed again from memory, so that the ordinary path holds nothing for this one.)
        const int keys = min(kKeys, bl.nk - n * kKeys);
        const int64_t t = bl.q0 + min(qi, bl.nq - 1);
        const uint16_t* qn = (const uint16_t*)a.q_nope + t * a.q_nope_token_stride + (int64_t)h * a.q_nope_head_stride;
        const uint16_t* qr = (const uint16_t*)a.q_rope + t * a.q_rope_token_stride + (int64_t)h * a.q_rope_head_stride;
        const float off = m == -__builtin_huge_valf() ? 0.0f : m;
#pragma unroll 1
        for (int j = 0; j < keys; j++) {
          const uint16_t* row = kv + (int64_t)(n * kKeys + j) * a.kv_token_stride;
          const uint16_t* rot = kr + (int64_t)(n * kKeys + j) * a.k_rope_stride;
          float score = 0.0f;
#pragma unroll 1
          for (int c = half; c < NC + PC; c += 2) {  // the other chunks are the pair's other lane's
            float x[8], y[8];
            unpack8<DT>(*(const uint4*)(c < NC ? qn + 8 * c : qr + 8 * (c - NC)), x);
            unpack8<DT>(*(const uint4*)(c < NC ? row + 8 * c : rot + 8 * (c - NC)), y);
#pragma unroll
            for (int i = 0; i < 8; i++) score = __builtin_fmaf(x[i], y[i], score);
          }
          score = a.scale < 0.0f ? -pair_sum(score) : pair_sum(score);
          const float e = __builtin_amdgcn_exp2f(__builtin_fmaf(score - off, scale, kProbShift<DT>));
          if (n * kKeys + j > limit) continue;
          const bool some = pack2<DT>(e, e) != 0;
          const uint16_t* x = row + N + 4 * half;
#pragma unroll
          for (int c = 0; c < VB; c++)
#pragma unroll
            for (int i = 0; i < 16; i++) {
              const uint16_t y = x[32 * c + 8 * (i >> 2) + (i & 3)];
              if (finite_only<DT>(y) != y) o[c][i] += some ? to_f32<DT>(y) : __builtin_nanf("");
            }
        }
      }
    }
    s[0] = s_next[0];
    s[1] = s_next[1];
  }

  if (qi >= bl.nq) return;
  l = pair_sum(l);
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  uint16_t* out = (uint16_t*)a.out + (int64_t)(bl.q0 + qi) * a.out_token_stride + (int64_t)h * a.out_head_stride;
#pragma unroll
  for (int c = 0; c < VB; c++)
#pragma unroll
    for (int i = 0; i < 16; i += 8) {
      // columns 8 (i / 4) + 4 half + 0..3 and 8 further: the pair of lanes trades halves, so that each has 8 neighbouring ones
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 2; j++) {
        const auto x = __builtin_amdgcn_permlane32_swap(pack2<DT>(o[c][i + 2 * j] * inv, o[c][i + 2 * j + 1] * inv),
                                                        pack2<DT>(o[c][i + 4 + 2 * j] * inv, o[c][i + 5 + 2 * j] * inv), false, false);
        w[j] = x[0];
        w[2 + j] = x[1];
      }
      *(uint4*)(out + 32 * c + 2 * i + 8 * half) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

template <int DT, int N, int P, int V>
int launch_prefill(const vib3_mla_prefill& a, hipStream_t st) {
  // Sequences' blocks number at most this many (each ends in one that is not full); surplus workgroups end at once. Measured with
  // 128 + 64 + 128 in bf16, us with 256 queries a workgroup / with 128 (one workgroup a CU in both forms):
  //   one prompt, by the count `wide`   128: 27 / 24 (500 tokens of 64 heads), 19 / 17 (256 of 128); 192: 33 / 34 (700 of 64), 108 / 100
  //                                     (3000 of 16); 240: 62 / 66 (1500 of 40); 256: 46 / 51 (1000 of 64); 512: 104 / 151 (2048 of 64)
  //   few queries over many keys        701 / 778 (32 of 1 query over 3000 keys, 64 heads), 118 / 130 (4 over 4000): twice the waves
  //                                     load the tiles
  //   one long prompt among others      131 / 121 (4096 tokens and 31 single queries, 8 heads): the host does not know the lengths,
  //                                     and takes the blocks that there may be
  // With 64 + 32 + 64 the forms are within 4 % of one another for one prompt to 2000 tokens, and 256 queries better by up to 10 %
  // (16 for 8 or 16 heads of 6000) beyond; many short sequences would be better off with 128 (502 / 331 for the 32 over 3000, 38 / 27
  // for 20 prompts of 100), of which two workgroups fit in a CU, four over 4000 keys not (85 / 105).
  const int64_t wide = (a.q_tokens + 255 * (int64_t)a.num_seqs) / 256 * a.heads;
  const int64_t narrow = (a.q_tokens + 127 * (int64_t)a.num_seqs) / 128 * a.heads;
  if (narrow > 0x7fffffff) return VIB3_ERR_BAD_COUNT;
  if (wide >= 224)  // of 256 CUs
    hipLaunchKernelGGL((k_mla_prefill<DT, N, P, V, 8>), dim3((unsigned)wide), dim3(512), 0, st, a);
  else
    hipLaunchKernelGGL((k_mla_prefill<DT, N, P, V, 4>), dim3((unsigned)narrow), dim3(256), 0, st, a);
  VIB3_RETURN_LAUNCH();
}

template <int DT, int N, int P>
int launch_prefill_v(const vib3_mla_prefill& a, hipStream_t st) {
  return a.v_dim == 128 ? launch_prefill<DT, N, P, 128>(a, st) : launch_prefill<DT, N, P, 64>(a, st);
}

template <int DT>
int launch_prefill_dt(const vib3_mla_prefill& a, hipStream_t st) {
  if (a.nope == 128) return a.rope == 64 ? launch_prefill_v<DT, 128, 64>(a, st) : launch_prefill_v<DT, 128, 32>(a, st);
  return a.rope == 64 ? launch_prefill_v<DT, 64, 64>(a, st) : launch_prefill_v<DT, 64, 32>(a, st);
}

}  // namespace vib3

using namespace vib3;

extern "C" int vib3_launch_mla_prefill(const vib3_mla_prefill* args, void* stream) {
  if (!args) return VIB3_ERR_BAD_POINTER;
  const vib3_mla_prefill& a = *args;
  if (!mla_dtype(a.dtype) || (a.nope != 64 && a.nope != 128) || (a.v_dim != 64 && a.v_dim != 128) ||
      (a.rope != 32 && a.rope != 64))
    return VIB3_ERR_UNSUPPORTED;
  if (!__builtin_isfinite(a.scale)) return VIB3_ERR_UNSUPPORTED;
  if (a.heads < 1 || a.heads > 65535 || a.num_seqs < 0 || a.q_tokens < 0 || a.k_tokens < 0) return VIB3_ERR_BAD_COUNT;
  if (a.q_tokens == 0 || a.num_seqs == 0) return 0;
  if (!a.cu_q || !a.cu_k || !mla_aligned(a.q_nope) || !mla_aligned(a.q_rope) || !mla_aligned(a.out) ||
      (a.k_tokens && (!mla_aligned(a.kv) || !mla_aligned(a.k_rope))) || !mla_stride(a.q_nope_token_stride) ||
      !mla_stride(a.q_nope_head_stride) || !mla_stride(a.q_rope_token_stride) || !mla_stride(a.q_rope_head_stride) ||
      !mla_stride(a.kv_token_stride) || !mla_stride(a.kv_head_stride) || !mla_stride(a.k_rope_stride) ||
      !mla_stride(a.out_token_stride) || !mla_stride(a.out_head_stride))
    return VIB3_ERR_BAD_POINTER;
  return a.dtype == VIB3_DT_F16 ? launch_prefill_dt<VIB3_DT_F16>(a, (hipStream_t)stream)
                                : launch_prefill_dt<VIB3_DT_BF16>(a, (hipStream_t)stream);
}
