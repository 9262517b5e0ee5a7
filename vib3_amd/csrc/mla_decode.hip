// mla_decode.hip — attention of single query tokens over the paged latent cache, absorbed form.
//
// Per row and head: ql = q_nope . W_uk, scores of every visible cached row against [ql | q_rope], softmax, the
// weighted sum of the latents, out = W_uv . that. All heads share the cached rows, so a row of 1152 bytes
// serves 64 heads x 2176 flops: at 64 heads the cache read and the matrix cores are of one order, and the read bounds.
// Three launches:
//   k_mla_absorb   ql for all rows, on the matrix cores; one more workgroup plans the next launch
//   k_mla_attend   the attention in the latent space, over equal shares of all rows' cached tokens
//   k_mla_finish   rows that several workgroups shared are joined, and W_uv applied
//
// The plan: tokens are taken 64 at a time (a unit), heads in groups of up to 64. All units of all items
// (row, head group) in order are cut into kShares equal runs, one workgroup each, whatever the rows' lengths: a long row is
// shared by many workgroups, a run covers many short rows. Nothing on the host depends on the lengths, so a captured
// launch follows them.
#include "mla.h"

namespace vib3 {

constexpr int kMlaMaxRows = 65536;
constexpr int kUnit = 64;      // cached tokens of one step
constexpr int kShares = 256;   // workgroups of the attention launch, one per CU (its LDS tiles fill one)
constexpr int kMinUnits = 1;   // units of a share at least

// Device workspace. Slot 2w holds the part of the item that share w starts in the middle of, or that it covers the
// middle of; slot 2w + 1 the part of the item it ends in (if it starts that item).
struct DecodeWs {
  int64_t* head;      // [2]: units per share, all units
  int64_t* prefix;    // [items + 1] units before each item
  int32_t* first;     // [kShares] item in which a share starts
  uint16_t* ql;       // [rows][heads][rank]
  uint16_t* ol;       // [rows][heads][rank] weighted latent of items that one share covers
  float* part;        // [2 kShares][heads of a group][rank] unnormalised sums
  float2* stat;       // [2 kShares][heads of a group] running maximum (of scores in log2 units) and sum
};

__host__ __device__ inline int head_groups(int heads) { return (heads + 63) / 64; }
__host__ __device__ inline int group_heads(int heads) { return heads < 64 ? heads : 64; }

inline size_t decode_ws(const vib3_mla_decode& a, DecodeWs* w, void* base) {
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t p = at;
    at += (bytes + 255) / 256 * 256;
    return (uint8_t*)base + p;
  };
  const size_t row = (size_t)a.heads * a.cache.rank;
  DecodeWs r;
  r.head = (int64_t*)take(16);
  r.prefix = (int64_t*)take(8 * ((size_t)a.rows * head_groups(a.heads) + 1));
  r.first = (int32_t*)take(4 * kShares);
  r.ql = (uint16_t*)take(a.kv_b ? 2 * row * a.rows : 0);
  r.ol = (uint16_t*)take(2 * row * a.rows);
  r.part = (float*)take(4 * (size_t)group_heads(a.heads) * a.cache.rank * 2 * kShares);
  r.stat = (float2*)take(8 * (size_t)group_heads(a.heads) * 2 * kShares);
  if (w) *w = r;
  return at;
}

struct DecodeArgs {
  vib3_mla_decode a;
  DecodeWs w;
};

// Visible cached tokens of row r and its sequence.
__device__ __forceinline__ int row_len(const vib3_mla_decode& a, int r, int* seq) {
  const int s = a.seqs ? a.seqs[r] : r;
  *seq = s;
  return (unsigned)s < (unsigned)a.cache.num_seqs ? clamp_len(a.cache, a.lens[r]) : 0;
}

// ------------------------------------------------------------------------- the plan

// One workgroup of 256: running sums of the items' units, the share size, and the item each share starts in.
__device__ void make_plan(const vib3_mla_decode& a, const DecodeWs& w) {
  __shared__ int64_t wave_total[4];
  const int tid = (int)threadIdx.x, lane = tid & 63;
  const int groups = head_groups(a.heads), items = a.rows * groups;
  int64_t before = 0;
  for (int x0 = 0; x0 < items; x0 += 256) {
    const int x = x0 + tid;
    int seq;
    const int64_t n = x < items ? ((int64_t)row_len(a, x / groups, &seq) + kUnit - 1) / kUnit : 0;
    int64_t sum = n;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int64_t up = __shfl_up(sum, d);
      if (lane >= d) sum += up;
    }
    if (lane == 63) wave_total[tid >> 6] = sum;
    __syncthreads();
    int64_t base = before;
    for (int i = 0; i < 4; i++) {
      if (i < (tid >> 6)) base += wave_total[i];
      before += wave_total[i];
    }
    if (x < items) w.prefix[x] = base + sum - n;
    __syncthreads();
  }
  const int64_t per = max((int64_t)kMinUnits, (before + kShares - 1) / kShares);
  if (tid == 0) {
    w.prefix[items] = before;
    w.head[0] = per;
    w.head[1] = before;
  }
  __syncthreads();
  for (int x = tid; x < items; x += 256) {
    const int64_t lo = w.prefix[x], hi = w.prefix[x + 1];
    for (int64_t s = (lo + per - 1) / per; s * per < hi; s++) w.first[s] = x;
  }
}

__global__ __launch_bounds__(256) void k_mla_plan(DecodeArgs d) { make_plan(d.a, d.w); }

// ------------------------------------------------------------------------- ql = q_nope . W_uk

constexpr int kAbsorbCols = 128;

// A workgroup takes 128 latent columns of one head: that part of W_uk goes to LDS once, and 16 rows at a
// time are multiplied by it as (W_uk^T) . (q^T), each wave 32 columns. W_uk lies with the latent columns contiguous, so
// its operand is read transposed. LDS rows are 256 bytes; 16-byte chunk c of row n lies at c ^ swizzle(n), which
// spreads a transposing read over the banks.
__device__ __forceinline__ int absorb_swizzle(int n) { return ((n & 3) << 2) ^ (((n >> 3) & 1) << 1); }

template <int DT>
__global__ __launch_bounds__(256) void k_mla_absorb(DecodeArgs d, int col_blocks) {
  const vib3_mla_decode& a = d.a;
  __shared__ __align__(16) uint8_t tile[256 * kAbsorbCols * 2];
  if ((int)blockIdx.x == a.heads * col_blocks) {
    if (blockIdx.y == 0) make_plan(a, d.w);
    return;
  }
  const int h = (int)blockIdx.x / col_blocks, c0 = ((int)blockIdx.x % col_blocks) * kAbsorbCols;
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int rank = a.cache.rank;
  const uint16_t* w = (const uint16_t*)a.kv_b + (size_t)h * (a.nope + a.v_dim) * rank + c0;
  for (int i = wave; i < a.nope / 4; i += 4) {  // four rows of W_uk at a time
    const int n = 4 * i + (lane >> 4), c = (lane & 15) ^ absorb_swizzle(n);
    load_to_lds16(w + (size_t)n * rank + 8 * c, (lds_u8*)tile + i * 1024);
  }
  const int row = lane & 15, g = lane >> 4;
  // this lane's element of a transposing read: row 8 g + row / 4 (+ 4), columns 16 blk + 4 (row % 4)
  const int n0 = 8 * g + (row >> 2);
  const int part = 8 * (row & 1);
  const int r_end = min(a.rows, ((int)blockIdx.y + 1) * 64);
  wait_lds_loads();
  __syncthreads();
  for (int r0 = (int)blockIdx.y * 64; r0 < r_end; r0 += 16) {
    const int r = min(r0 + row, a.rows - 1);
    const uint16_t* q = (const uint16_t*)a.q_nope + (int64_t)r * a.q_nope_row_stride + (int64_t)h * a.q_nope_head_stride;
    f32x4 acc[2] = {};
    for (int k = 0; k < a.nope; k += 32) {
      const s16x8 b = *(const s16x8*)(q + k + 8 * g);
#pragma unroll
      for (int blk = 0; blk < 2; blk++) {
        const int c = (wave * 2 + blk) * 2 + ((row & 3) >> 1);
        const int na = k + n0, nb = na + 4;
        const s16x4 lo = lds_read_tr((lds_u8*)tile + na * 256 + (c ^ absorb_swizzle(na)) * 16 + part);
        const s16x4 hi = lds_read_tr((lds_u8*)tile + nb * 256 + (c ^ absorb_swizzle(nb)) * 16 + part);
        acc[blk] = mma32<DT>(join(lo, hi), b, acc[blk]);
      }
    }
    if (r0 + row < a.rows) {
      uint16_t* o = d.w.ql + ((size_t)(r0 + row) * a.heads + h) * rank + c0 + wave * 32 + 4 * g;
#pragma unroll
      for (int blk = 0; blk < 2; blk++)  // rounded for the matrix cores: relative error half a step
        *(uint2*)(o + 16 * blk) = make_uint2(pack2<DT>(acc[blk][0], acc[blk][1]), pack2<DT>(acc[blk][2], acc[blk][3]));
    }
  }
}

// ------------------------------------------------------------------------- attention in the latent space

// What masked tokens read instead of the cache: their probability is 0, and 0 times whatever lies there must be 0.
__device__ const uint4 zero_row[(512 + 64) / 8] = {};

// A workgroup is eight waves, two per SIMD, and takes HB blocks of 16 heads (1, 2 or 4; more than 64 heads are groups of 64,
// planned like rows of their own). For a unit of 64 tokens it forms the scores S^T = K . Q^T, the waves dealt over
// (head block, 16 tokens), so that a lane holds one head's scores of 4 tokens; the running maximum of a head over
// the unit is joined through LDS; the probabilities go to LDS, and each wave adds to the sums O^T = C^T . P^T of all heads for an
// eighth of the latent's columns, C^T by transposing reads of the same LDS rows. Splitting the columns keeps a
// wave's sums at 64 registers (heads x 64 columns), so that next to the 72 of its queries enough remain for LDS reads in
// flight, and every cached row is read from LDS once for all heads' sums.
//
// A unit's rows go from the pages straight to LDS (16 bytes a lane), double-buffered: while one unit is
// worked on, the next is in flight (74 KB a CU, 19 MB over the chip). A row's 16-byte chunk c lies at c ^ f(row)
// (f = (row / 2) % 8, rows 32 banks apart; for widths of 4 chunks modulo 8 (row / 4) % 4, rows 16 banks apart), which
// spreads the row-wise and the transposing reads over all 64 banks.
template <int DT, int R, int P, int HB>
__global__ __launch_bounds__(512, 2) void k_mla_attend(DecodeArgs d) {
  constexpr int kWaves = 8;
  constexpr int W = R + P, CH = W / 8, kRowBytes = W * 2;
  constexpr int kMask = CH % 8 == 0 ? 7 : 3, kShift = CH % 8 == 0 ? 1 : 2;
  constexpr int kTpw = kUnit / kWaves;                 // rows a wave loads
  constexpr int kLoads = (kTpw * CH + 63) / 64;
  constexpr int kTile = kUnit * kRowBytes;
  constexpr int NB = HB == 4 ? 2 : 1;                  // 16-token blocks of a wave's scores (HB = 1: four waves have none)
  constexpr int CB = R / 16 / kWaves;                  // 16-column blocks of a wave's sums
  __shared__ __align__(1024) uint8_t tile[2 * kTile];
  __shared__ __align__(16) uint8_t prob[HB * 16 * kUnit * 2];  // [head][token], chunk c of a row at c ^ (head / 2) % 8
  __shared__ float tops[4][HB * 16];                   // maximum of 16 tokens' scores per head; at the end their sums
  __shared__ float fade[HB * 16];                      // factor of a head's earlier sums
  __shared__ float2 stats[HB * 16];                    // at the end: maximum and sum
  __shared__ __align__(16) float seen[2][kUnit];       // 1: the token is seen
  __shared__ uint64_t row_at[kUnit];                   // addresses of the next unit's rows, each wave its own

  const vib3_mla_decode& a = d.a;
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int g = lane >> 4, col = lane & 15;
  // this wave's scores: head block hb, token blocks tb .. tb + NB - 1
  const int hb = HB == 4 ? wave >> 1 : HB == 2 ? wave >> 2 : 0;
  const int tb = HB == 4 ? (wave & 1) * 2 : wave & 3;
  const bool scores = HB > 1 || wave < 4;
  const int groups = head_groups(a.heads);
  const float to_log2 = a.scale * 1.44269504088896341f;

  const int64_t per = d.w.head[0], all = d.w.head[1];
  const int64_t begin = (int64_t)blockIdx.x * per, end = min(begin + per, all);
  if (begin >= end) return;
  int x = d.w.first[blockIdx.x];

  // this lane's places within a tile: row tb * 16 + col for the scores, row 8 g + col / 4 (and 4 further) for the transposing
  // reads, at 16 * wave * CB columns; 16 rows further the swizzle is the same
  const int krow = tb * 16 + col, kf = (krow >> kShift) & kMask;
  const int vrow = 8 * g + (col >> 2), vf0 = (vrow >> kShift) & kMask, vf1 = ((vrow + 4) >> kShift) & kMask;
  lds_u8* const pw = (lds_u8*)prob + (hb * 16 + col) * (kUnit * 2);  // where this lane's probabilities go
  const int pf = (col >> 1) & 7;

  for (int64_t u0 = begin; u0 < end; x++) {
    const int64_t row_begin = d.w.prefix[x], row_end = d.w.prefix[x + 1];
    const int64_t u1 = min(end, row_end);
    if (u1 <= u0) continue;
    const int r = x / groups, h0 = (x - r * groups) * 64;
    int seq;
    const int len = row_len(a, r, &seq);
    const int32_t* table = a.cache.block_table + (size_t)seq * a.cache.max_pages;
    const int first_unit = (int)(u0 - row_begin), units = (int)(u1 - u0);

    // token of unit n whose row this lane finds the address of (lanes < kTpw), and its page's number
    auto page_of = [&](int n) {
      const int j = (first_unit + n) * kUnit + wave * kTpw + lane;
      return lane < kTpw && n < units && j < len ? table[j / a.cache.page_size] : -1;
    };
    auto issue = [&](int n, int id) {
      const int j = (first_unit + n) * kUnit + wave * kTpw + lane;
      const bool ok = (unsigned)id < (unsigned)a.cache.num_pages;
      const uint16_t* p = (const uint16_t*)zero_row;
      if (ok)
        p = (const uint16_t*)a.cache.pool + (int64_t)id * a.cache.page_stride +
            (int64_t)(j % a.cache.page_size) * a.cache.row_stride;
      if (lane < kTpw) {
        seen[n & 1][wave * kTpw + lane] = ok ? 1.0f : 0.0f;
        row_at[wave * kTpw + lane] = (uint64_t)(uintptr_t)p;
      }
      lds_u8* base = (lds_u8*)tile + (n & 1) * kTile + wave * kTpw * kRowBytes;
      int ln = lane;
      asm volatile("" : "+v"(ln));  // the loads' places are formed anew for each unit, not held in registers
#pragma unroll
      for (int i = 0; i < kLoads; i++) {
        const int slot = i * 64 + ln, t = slot / CH;
        const int c = (slot - t * CH) ^ (((wave * kTpw + t) >> kShift) & kMask);
        if (kTpw * CH % 64 == 0 || slot < kTpw * CH)
          load_to_lds16((const uint8_t*)(uintptr_t)row_at[wave * kTpw + t] + c * 16, base + i * 1024);
      }
    };

    // queries: the B operand, this lane's head at k = 32 s + 8 g
    s16x8 q[W / 32];
    {
      const int64_t hh = min(h0 + hb * 16 + col, a.heads - 1);
      const uint16_t* ql = a.kv_b ? d.w.ql + ((size_t)r * a.heads + hh) * R
                                  : (const uint16_t*)a.q_nope + r * a.q_nope_row_stride + hh * a.q_nope_head_stride;
      const uint16_t* qr = (const uint16_t*)a.q_rope + r * a.q_rope_row_stride + hh * a.q_rope_head_stride;
#pragma unroll
      for (int s = 0; s < W / 32; s++) q[s] = *(const s16x8*)(s < R / 32 ? ql + 32 * s + 8 * g : qr + 32 * (s - R / 32) + 8 * g);
    }
    f32x4 o[HB][CB] = {};
    float m = -__builtin_huge_valf(), l = 0.0f;  // of this lane's head; l over this lane's own tokens

    int id = page_of(0);
    __syncthreads();  // the last item's tiles and statistics are done with
    issue(0, id);
    id = page_of(1);
    for (int n = 0; n < units; n++) {
      wait_lds_loads();
      __syncthreads();  // unit n is in LDS; everyone is past unit n - 1
      if (n + 1 < units) {
        issue(n + 1, id);
        id = page_of(n + 2);
      }
      lds_u8* t = (lds_u8*)tile + (n & 1) * kTile;
      f32x4 s[NB] = {};
      if (scores) {
#pragma unroll
        for (int k = 0; k < W / 32; k++) {
          const int c = ((4 * k + g) & ~kMask) | (((4 * k + g) & kMask) ^ kf);
#pragma unroll
          for (int b = 0; b < NB; b++) s[b] = mma32<DT>(lds_read16(t + (krow + 16 * b) * kRowBytes + c * 16), q[k], s[b]);
        }
#pragma unroll
        for (int b = 0; b < NB; b++) {
          const float4 v = *(const float4*)&seen[n & 1][(tb + b) * 16 + 4 * g];
          const float vv[4] = {v.x, v.y, v.z, v.w};
          float top = -__builtin_huge_valf();
#pragma unroll
          for (int i = 0; i < 4; i++) {
            s[b][i] = vv[i] != 0.0f ? s[b][i] * to_log2 : -__builtin_huge_valf();
            top = fmaxf(top, s[b][i]);
          }
          top = fmaxf(top, __shfl_xor(top, 16));
          top = fmaxf(top, __shfl_xor(top, 32));
          if (g == 0) tops[tb + b][hb * 16 + col] = top;
        }
      }
      __syncthreads();
      if (scores) {
        const int at = hb * 16 + col;
        const float mn = fmaxf(m, fmaxf(fmaxf(tops[0][at], tops[1][at]), fmaxf(tops[2][at], tops[3][at])));
        const float base = mn == -__builtin_huge_valf() ? 0.0f : mn;
        const float f = __builtin_amdgcn_exp2f(m - base);
        m = mn;
        l *= f;
        if (g == 0 && tb == 0) fade[at] = f;
#pragma unroll
        for (int b = 0; b < NB; b++) {
          float e[4];
#pragma unroll
          for (int i = 0; i < 4; i++) {
            e[i] = __builtin_amdgcn_exp2f(s[b][i] - base);
            l += e[i];
          }
          // rounded for the matrix cores; the sum l takes them unrounded
          lds_write8(pw + ((2 * (tb + b) + (g >> 1)) ^ pf) * 16 + 8 * (g & 1), pack2<DT>(e[0], e[1]), pack2<DT>(e[2], e[3]));
        }
      }
      __syncthreads();
#pragma unroll
      for (int h = 0; h < HB; h++) {
        const float f = fade[h * 16 + col];
        if (__any(f != 1.0f)) {
#pragma unroll
          for (int c = 0; c < CB; c++) o[h][c] *= f;
        }
      }
#pragma unroll
      for (int k = 0; k < kUnit / 32; k++) {
        s16x8 pb[HB];
#pragma unroll
        for (int h = 0; h < HB; h++)
          pb[h] = lds_read16((lds_u8*)prob + (h * 16 + col) * (kUnit * 2) + ((4 * k + g) ^ pf) * 16);
#pragma unroll
        for (int c = 0; c < CB; c++) {
          const int ch = 2 * (wave * CB + c) + ((col & 3) >> 1);
          lds_u8* v = t + (32 * k + vrow) * kRowBytes + 8 * (col & 1);
          const s16x8 av = join(lds_read_tr(v + ((ch & ~kMask) | ((ch & kMask) ^ vf0)) * 16),
                                lds_read_tr(v + 4 * kRowBytes + ((ch & ~kMask) | ((ch & kMask) ^ vf1)) * 16));
#pragma unroll
          for (int h = 0; h < HB; h++) o[h][c] = mma32<DT>(av, pb[h], o[h][c]);
        }
      }
    }
    // the heads' sums of probabilities, over a wave's lanes and the waves of a head block
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    __syncthreads();
    if (scores && g == 0) {
      tops[HB == 4 ? tb >> 1 : tb][hb * 16 + col] = l;
      if (tb == 0) stats[hb * 16 + col].x = m;
    }
    __syncthreads();
    const bool whole = u0 == row_begin && u1 == row_end;
#pragma unroll
    for (int h = 0; h < HB; h++) {
      const int at = h * 16 + col, head = h0 + at;
      const float sum = HB == 4 ? tops[0][at] + tops[1][at] : (tops[0][at] + tops[1][at]) + (tops[2][at] + tops[3][at]);
      if (head >= a.heads) continue;
      const int c0 = wave * CB * 16 + 4 * g;
      if (whole) {
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        uint16_t* out = d.w.ol + ((size_t)r * a.heads + head) * R + c0;
#pragma unroll
        for (int c = 0; c < CB; c++)
          *(uint2*)(out + 16 * c) =
              make_uint2(pack2<DT>(o[h][c][0] * inv, o[h][c][1] * inv), pack2<DT>(o[h][c][2] * inv, o[h][c][3] * inv));
      } else {
        const size_t slot = (2 * (size_t)blockIdx.x + (u0 == begin ? 0 : 1)) * group_heads(a.heads) + at;
        float* out = d.w.part + slot * R + c0;
#pragma unroll
        for (int c = 0; c < CB; c++) *(float4*)(out + 16 * c) = make_float4(o[h][c][0], o[h][c][1], o[h][c][2], o[h][c][3]);
        if (g == 0 && wave == 0) d.w.stat[slot] = make_float2(stats[at].x, sum);
      }
    }
    u0 = u1;
  }
}

// ------------------------------------------------------------------------- joined rows and W_uv

// A workgroup takes 16 rows of one head: their weighted latents (joined from the shares' parts where a row
// has several) go to LDS in 16 bits, and each wave multiplies them by 16 rows of W_uv at a time. Without W_uv
// the weighted latents are the result.
template <int DT, int R>
__global__ __launch_bounds__(256) void k_mla_finish(DecodeArgs d) {
  const vib3_mla_decode& a = d.a;
  constexpr int kStride = R + 8;  // 16 bytes more: rows start in different banks
  __shared__ __align__(16) uint16_t lat[16 * kStride];
  const int h = (int)blockIdx.x, r0 = (int)blockIdx.y * 16;
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t per = d.w.head[0];
  constexpr int kCols = R / 64;  // columns of a lane: one wave joins a row
  for (int i = wave; i < 16; i += 4) {
    const int r = r0 + i;
    uint16_t* dst = lat + i * kStride + lane * kCols;
    float o[kCols] = {};
    const int x = r * head_groups(a.heads) + h / 64;
    const int64_t lo = r < a.rows ? d.w.prefix[x] : 0, hi = r < a.rows ? d.w.prefix[x + 1] : 0;
    if (hi > lo) {
      const int64_t w0 = lo / per, w1 = (hi - 1) / per;
      if (w0 == w1) {
        const uint16_t* p = d.w.ol + ((size_t)r * a.heads + h) * R + lane * kCols;
#pragma unroll
        for (int c = 0; c < kCols; c++) o[c] = to_f32<DT>(p[c]);
      } else {
        float m = -__builtin_huge_valf(), l = 0.0f;
        for (int64_t w = w0; w <= w1; w++) {
          const size_t at = (2 * (size_t)w + (w == w0 && lo != w * per ? 1 : 0)) * group_heads(a.heads) + h % 64;
          const float2 s = d.w.stat[at];
          const float* p = d.w.part + at * R + lane * kCols;
          const float mn = fmaxf(m, s.x), base = mn == -__builtin_huge_valf() ? 0.0f : mn;
          const float f0 = __builtin_amdgcn_exp2f(m - base), f1 = __builtin_amdgcn_exp2f(s.x - base);
          l = l * f0 + s.y * f1;
#pragma unroll
          for (int c = 0; c < kCols; c++) o[c] = o[c] * f0 + p[c] * f1;
          m = mn;
        }
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
        for (int c = 0; c < kCols; c++) o[c] *= inv;
      }
    }
    if (a.kv_b) {
#pragma unroll
      for (int c = 0; c < kCols; c++) dst[c] = from_f32<DT>(o[c]);
    } else if (r < a.rows) {
      uint16_t* out = (uint16_t*)a.out + (int64_t)r * a.out_row_stride + (int64_t)h * a.out_head_stride + lane * kCols;
#pragma unroll
      for (int c = 0; c < kCols; c++) out[c] = from_f32<DT>(o[c]);
    }
  }
  if (!a.kv_b) return;
  __syncthreads();
  const int g = lane >> 4, n = lane & 15;
  for (int v0 = wave * 16; v0 < a.v_dim; v0 += 64) {
    const uint16_t* w = (const uint16_t*)a.kv_b + ((size_t)h * (a.nope + a.v_dim) + a.nope + v0 + n) * R;
    f32x4 acc = {};
#pragma unroll
    for (int k = 0; k < R; k += 32)  // rows of W_uv times the rows' latents: a lane ends with 4 outputs of one row
      acc = mma32<DT>(*(const s16x8*)(w + k + 8 * g), *(const s16x8*)(lat + n * kStride + k + 8 * g), acc);
    const int r = r0 + n;
    if (r < a.rows)
      *(uint2*)((uint16_t*)a.out + (int64_t)r * a.out_row_stride + (int64_t)h * a.out_head_stride + v0 + 4 * g) =
          make_uint2(pack2<DT>(acc[0], acc[1]), pack2<DT>(acc[2], acc[3]));
  }
}

template <int DT, int R, int P>
int launch_decode(const DecodeArgs& d, hipStream_t st) {
  const vib3_mla_decode& a = d.a;
  if (a.kv_b) {
    const int col_blocks = R / kAbsorbCols;
    hipLaunchKernelGGL(k_mla_absorb<DT>, dim3((unsigned)(a.heads * col_blocks + 1), (unsigned)((a.rows + 63) / 64)), dim3(256), 0, st,
                       d, col_blocks);
  } else {
    hipLaunchKernelGGL(k_mla_plan, dim3(1), dim3(256), 0, st, d);
  }
  if (a.heads <= 16)
    hipLaunchKernelGGL((k_mla_attend<DT, R, P, 1>), dim3(kShares), dim3(512), 0, st, d);
  else if (a.heads <= 32)
    hipLaunchKernelGGL((k_mla_attend<DT, R, P, 2>), dim3(kShares), dim3(512), 0, st, d);
  else
    hipLaunchKernelGGL((k_mla_attend<DT, R, P, 4>), dim3(kShares), dim3(512), 0, st, d);
  hipLaunchKernelGGL((k_mla_finish<DT, R>), dim3((unsigned)a.heads, (unsigned)((a.rows + 15) / 16)), dim3(256), 0, st, d);
  VIB3_RETURN_LAUNCH();
}

template <int DT>
int launch_decode_dt(const DecodeArgs& d, hipStream_t st) {
  if (d.a.cache.rank == 512)
    return d.a.cache.rope == 64 ? launch_decode<DT, 512, 64>(d, st) : launch_decode<DT, 512, 32>(d, st);
  return d.a.cache.rope == 64 ? launch_decode<DT, 256, 64>(d, st) : launch_decode<DT, 256, 32>(d, st);
}

bool decode_counts(const vib3_mla_decode& a) {
  return a.rows >= 0 && a.rows <= kMlaMaxRows && a.heads >= 1 && a.heads <= 128;
}

}  // namespace vib3

using namespace vib3;

extern "C" size_t vib3_mla_decode_workspace_bytes(const vib3_mla_decode* args) {
  if (!args || !decode_counts(*args) || (args->cache.rank != 256 && args->cache.rank != 512)) return 0;
  vib3_mla_decode a = *args;
  a.kv_b = &a;  // the larger of the two forms
  return decode_ws(a, nullptr, nullptr);
}

extern "C" int vib3_launch_mla_decode(const vib3_mla_decode* args, void* stream) {
  if (!args) return VIB3_ERR_BAD_POINTER;
  const vib3_mla_decode& a = *args;
  if (const int rc = check_cache(a.cache)) return rc;
  if (!decode_counts(a)) return VIB3_ERR_BAD_COUNT;
  if (a.kv_b && (a.nope < 32 || a.nope > 256 || a.nope % 32 || a.v_dim < 32 || a.v_dim > 256 || a.v_dim % 32))
    return VIB3_ERR_UNSUPPORTED;
  if (a.rows == 0) return 0;
  if (!a.lens || !mla_aligned(a.q_nope) || !mla_aligned(a.q_rope) || !mla_aligned(a.out) ||
      (a.kv_b && !mla_aligned(a.kv_b)) || !mla_stride(a.q_nope_row_stride) || !mla_stride(a.q_nope_head_stride) ||
      !mla_stride(a.q_rope_row_stride) || !mla_stride(a.q_rope_head_stride) || !mla_stride(a.out_row_stride) ||
      !mla_stride(a.out_head_stride) || !a.workspace || ((uintptr_t)a.workspace & 255))
    return VIB3_ERR_BAD_POINTER;
  if (a.workspace_bytes < vib3_mla_decode_workspace_bytes(args)) return VIB3_ERR_WORKSPACE;
  DecodeArgs d;
  d.a = a;
  decode_ws(a, &d.w, a.workspace);
  return a.cache.dtype == VIB3_DT_F16 ? launch_decode_dt<VIB3_DT_F16>(d, (hipStream_t)stream)
                                      : launch_decode_dt<VIB3_DT_BF16>(d, (hipStream_t)stream);
}
