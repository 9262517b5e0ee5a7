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
struct Item {
  int64_t begin;      // units before the item
  int32_t len, seq;   // visible tokens of its row, and their sequence
};

struct Share {        // what a workgroup starts with
  int64_t total;      // its units
  int32_t item, seq, len, unit, left;  // the first item, its units before the share and in it
  int32_t pad;
};

struct DecodeWs {
  int64_t* head;      // [2]: units per share, all units
  Item* items;        // [items + 1]
  Share* shares;      // [kShares]
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
  r.items = (Item*)take(sizeof(Item) * ((size_t)a.rows * head_groups(a.heads) + 1));
  r.shares = (Share*)take(sizeof(Share) * kShares);
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
    int seq = 0;
    const int len = x < items ? row_len(a, x / groups, &seq) : 0;
    const int64_t n = ((int64_t)len + kUnit - 1) / kUnit;
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
    if (x < items) w.items[x] = Item{base + sum - n, len, seq};
    __syncthreads();
  }
  const int64_t per = max((int64_t)kMinUnits, (before + kShares - 1) / kShares);
  if (tid == 0) {
    w.items[items] = Item{before, 0, 0};
    w.head[0] = per;
    w.head[1] = before;
  }
  __syncthreads();
  static_assert(kShares == 256, "a thread per share");
  const int64_t from = tid * per, to = min(from + per, before);
  if (from >= before) {
    w.shares[tid].total = 0;
    return;
  }
  int lo = 0, hi = items;  // the last item that begins at or before the share's first unit: the one that holds it
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (w.items[mid].begin <= from) lo = mid;
    else hi = mid;
  }
  const Item it = w.items[lo];
  w.shares[tid] = Share{to - from, lo, it.seq, it.len, (int32_t)(from - it.begin),
                        (int32_t)(min(to, w.items[lo + 1].begin) - from), 0};
}

__global__ __launch_bounds__(256) void k_mla_plan(DecodeArgs d) { make_plan(d.a, d.w); }

// ------------------------------------------------------------------------- ql = q_nope . W_uk

constexpr int kAbsorbCols = 128;
constexpr int kAbsorbRows = 64;

// A workgroup takes 128 latent columns of one head for 64 rows, 16 rows a wave: that part of W_uk goes to LDS while each wave loads
// its queries, and is multiplied as (W_uk^T) . (q^T). W_uk lies with the latent columns contiguous, so its operand is read
// transposed. LDS rows are 256 bytes; 16-byte chunk c of row n lies at c ^ swizzle(n), which spreads a transposing read over the
// banks. Bound by the read of W_uk (8.4 MB for 64 heads of 128 x 512), and below some 16 rows by its latency.
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
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rank = a.cache.rank;
  const uint16_t* w = (const uint16_t*)a.kv_b + (size_t)h * (a.nope + a.v_dim) * rank + c0;
  for (int i = wave; i < a.nope / 4; i += 4) {  // four rows of W_uk at a time
    const int n = 4 * i + (lane >> 4), c = (lane & 15) ^ absorb_swizzle(n);
    load_to_lds16(w + (size_t)n * rank + 8 * c, (lds_u8*)tile + i * 1024);
  }
  const int row = lane & 15, g = lane >> 4;
  const int r = (int)blockIdx.y * kAbsorbRows + wave * 16 + row;
  const uint16_t* q = (const uint16_t*)a.q_nope + (int64_t)min(r, a.rows - 1) * a.q_nope_row_stride + (int64_t)h * a.q_nope_head_stride + 8 * g;
  s16x8 b[8];
#pragma unroll
  for (int k = 0; k < 8; k++) b[k] = k * 32 < a.nope ? *(const s16x8*)(q + k * 32) : s16x8{};
  // this lane's element of a transposing read: row 8 g + row / 4 (+ 4), columns 16 blk + 4 (row % 4)
  const int n0 = 8 * g + (row >> 2);
  wait_lds_loads();
  __syncthreads();
  if ((int)blockIdx.y * kAbsorbRows + wave * 16 >= a.rows) return;
  f32x4 acc[8] = {};
#pragma unroll
  for (int k = 0; k < 8; k++) {
    if (k * 32 >= a.nope) break;
    const int na = k * 32 + n0, nb = na + 4;
    lds_u8* t = (lds_u8*)tile + na * 256 + 8 * (row & 1);
#pragma unroll
    for (int blk = 0; blk < 8; blk++) {
      const int c = blk * 2 + ((row & 3) >> 1);
      acc[blk] = mma32<DT>(join(lds_read_tr(t + (c ^ absorb_swizzle(na)) * 16), lds_read_tr(t + 1024 + (c ^ absorb_swizzle(nb)) * 16)),
                           b[k], acc[blk]);
    }
  }
  if (r < a.rows) {
    uint16_t* o = d.w.ql + ((size_t)r * a.heads + h) * rank + c0 + 4 * g;
#pragma unroll
    for (int blk = 0; blk < 8; blk++)  // rounded for the matrix cores: relative error half a step
      *(uint2*)(o + 16 * blk) = make_uint2(pack2<DT>(acc[blk][0], acc[blk][1]), pack2<DT>(acc[blk][2], acc[blk][3]));
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
// Rows go from the pages straight to LDS (16 bytes a lane), double-buffered: while a unit is worked on, the next, of
// this item or the share's next one, is in flight (74 KB a CU, 19 MB over the chip). The latent parts of the rows and the rotary parts lie apart, so
// that one load instruction covers whole rows. Chunk c (16 bytes) of a latent part lies at c ^ row_swizzle(row): the
// rows' stride is a multiple of all 64 banks, and so the 16 rows of a score operand, and the 8 rows of half a transposing
// read, fall into different banks; a rotary part has 128 bytes whatever its width, chunk c at c ^ (row / 2) % 8.
__device__ __forceinline__ int row_swizzle(int row) { return ((row & 3) << 1) | (((row >> 3) & 1) << 3) | ((row >> 2) & 1); }

template <typename T>
__device__ __forceinline__ T ld_const(const T* p) {  // wave-uniform address: a scalar load
  return *(const __attribute__((address_space(4))) T*)p;
}

__device__ __forceinline__ const uint8_t* lane_ptr(uint64_t p, int lane) {  // a lane's pointer, wave-uniform
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)p, lane);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(p >> 32), lane);
  return (const uint8_t*)(uintptr_t)(((uint64_t)hi << 32) | lo);
}

// Maximum over the four lanes that share lane % 16.
__device__ __forceinline__ float max_over_rows(float v) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

template <int DT, int R, int P, int HB>
__global__ __launch_bounds__(512, 2) void k_mla_attend(DecodeArgs d) {
  constexpr int kWaves = 8;
  constexpr int kTpw = kUnit / kWaves;                 // rows a wave loads: 8, eight lanes for each
  constexpr int RC = R / 8, PC = P / 8;                // 16-byte chunks of the two parts of a row
  constexpr int kPer = 64 / RC;                        // latent parts of one load instruction: 1 or 2
  constexpr int NB = HB == 4 ? 2 : 1;                  // 16-token blocks of a wave's scores (HB = 1: four waves have none)
  constexpr int CB = R / 16 / kWaves;                  // 16-column blocks of a wave's sums
  __shared__ __align__(1024) uint8_t lat[2][kUnit * R * 2];
  __shared__ __align__(1024) uint8_t rot[2][kUnit * 128];
  __shared__ __align__(16) uint8_t prob[HB * 16 * kUnit * 2];  // [head][token], chunk c of a row at c ^ (head / 2) % 8
  __shared__ float tops[4][HB * 16];                   // maximum of 16 tokens' scores per head; at the end their sums
  __shared__ float fade[HB * 16];                      // factor of a head's earlier sums
  __shared__ float last_top[HB * 16];                  // at the end: the heads' maxima
  __shared__ __align__(16) float seen[2][kUnit];       // 1: the token is seen

  const vib3_mla_decode& a = d.a;
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, col = lane & 15;
  // this wave's scores: head block hb, token blocks tb .. tb + NB - 1
  const int hb = HB == 4 ? wave >> 1 : HB == 2 ? wave >> 2 : 0;
  const int tb = HB == 4 ? (wave & 1) * 2 : wave & 3;
  const bool scores = HB > 1 || wave < 4;
  const int groups = head_groups(a.heads);
  const float to_log2 = a.scale * 1.44269504088896341f;

  const Share* sh = d.w.shares + blockIdx.x;
  int64_t to_load = ld_const(&sh->total);  // units of the share not yet on their way to LDS
  if (to_load == 0) return;

  // The stream of units into LDS. Lane holds the token, page and place in the page of row wave * 8 + lane / 8 of the next unit to
  // look up, and the page's number and place of the next unit to load (-1: not seen).
  const int page_size = a.cache.page_size, page_step = kUnit / page_size, off_step = kUnit % page_size;
  int s_item = ld_const(&sh->item), s_left = ld_const(&sh->left), s_len = ld_const(&sh->len);  // of the unit to look up
  int64_t s_ahead = to_load;                                                                   // units not yet looked up
  const int32_t* s_table = a.cache.block_table + (size_t)ld_const(&sh->seq) * a.cache.max_pages;
  int s_token = ld_const(&sh->unit) * kUnit + wave * kTpw + (lane >> 3);
  int s_page = s_token / page_size, s_off = s_token - s_page * page_size;
  int id = -1, id_off = 0;
  auto look_up = [&] {
    if (s_left == 0 && s_ahead > 0) {
      int units;
      do {
        s_item++;
        s_len = ld_const(&d.w.items[s_item].len);
        units = (s_len + kUnit - 1) / kUnit;
      } while (units == 0);
      s_left = (int)min((int64_t)units, s_ahead);
      s_table = a.cache.block_table + (size_t)ld_const(&d.w.items[s_item].seq) * a.cache.max_pages;
      s_token = wave * kTpw + (lane >> 3);
      s_page = s_token / page_size;
      s_off = s_token - s_page * page_size;
    }
    id = -1;
    if (s_left > 0 && s_token < s_len) id = s_table[s_page];
    id_off = s_off;
    s_left--;
    s_ahead--;
    s_token += kUnit;
    s_off += off_step;
    s_page += page_step;
    if (s_off >= page_size) {
      s_off -= page_size;
      s_page++;
    }
  };
  auto issue = [&](int slot) {
    const bool ok = (unsigned)id < (unsigned)a.cache.num_pages;
    const uint64_t row = ok ? (uint64_t)(uintptr_t)((const uint16_t*)a.cache.pool + (int64_t)id * a.cache.page_stride +
                                                    (int64_t)id_off * a.cache.row_stride)
                            : (uint64_t)(uintptr_t)zero_row;
    const int ln = fresh(lane);
    if ((ln & 7) == 0) seen[slot][wave * kTpw + (ln >> 3)] = ok ? 1.0f : 0.0f;
#pragma unroll
    for (int i = 0; i < kTpw / kPer; i++) {
      const int t = i * kPer + (kPer == 2 ? ln >> 5 : 0);
      const uint8_t* p = lane_ptr(row, 8 * i * kPer);
      if (kPer == 2) {
        const uint8_t* p1 = lane_ptr(row, 8 * i * kPer + 8);
        p = ln >= 32 ? p1 : p;
      }
      load_to_lds16(p + ((ln & (RC - 1)) ^ row_swizzle(wave * kTpw + t)) * 16, (lds_u8*)lat[slot] + (wave * kTpw + i * kPer) * R * 2);
    }
    const int c = (ln & 7) ^ ((ln >> 4) & 3) ^ (wave & 1) * 4;  // (row / 2) % 8 of row wave * 8 + lane / 8
    if (PC == 8 || c < PC) load_to_lds16((const uint8_t*)(uintptr_t)row + R * 2 + c * 16, (lds_u8*)rot[slot] + wave * kTpw * 128);
  };

  // queries: the B operand, this lane's head at k = 32 s + 8 g
  s16x8 q[(R + P) / 32];
  auto load_q = [&](int x) {
    const int r = x / groups, h0 = (x - r * groups) * 64;
    const int64_t hh = min(h0 + hb * 16 + col, a.heads - 1);
    const uint16_t* ql = a.kv_b ? d.w.ql + ((size_t)r * a.heads + hh) * R
                                : (const uint16_t*)a.q_nope + r * a.q_nope_row_stride + hh * a.q_nope_head_stride;
    const uint16_t* qr = (const uint16_t*)a.q_rope + r * a.q_rope_row_stride + hh * a.q_rope_head_stride;
#pragma unroll
    for (int s = 0; s < (R + P) / 32; s++)
      q[s] = *(const s16x8*)(s < R / 32 ? ql + 32 * s + 8 * g : qr + 32 * (s - R / 32) + 8 * g);
  };

  // this lane's places within a unit: row tb * 16 + col for the scores, rows 8 g + col / 4 (and 4 further) for the
  // transposing reads; 16 rows further the swizzles are the same
  const int krow = tb * 16 + col, kf = row_swizzle(krow), rf = (col >> 1) & 7;
  const int vrow = 8 * g + (col >> 2), vf = row_swizzle(vrow);  // row_swizzle(vrow + 4) = vf | 1
  const int pf = (col >> 1) & 7;

  look_up();
  int x = ld_const(&sh->item), unit = ld_const(&sh->unit), units = ld_const(&sh->left), len = ld_const(&sh->len);
  int64_t left = to_load;
  issue(0);
  look_up();
  to_load--;
  load_q(x);
  VIB3_WAIT_VM(0);
  int n = 0;  // unit of the share
  for (;;) {
    f32x4 o[HB][CB] = {};
    float m = -__builtin_huge_valf(), l = 0.0f;  // of this lane's head; l over this lane's own tokens
    const int first_of_share = n;
    left -= units;
    int next = x;
    for (int i = 1;; i++, n++) {
      wait_lds_loads();
      __syncthreads();  // unit n is in LDS; everyone is done with unit n - 1
      if (to_load > 0) {
        issue((n + 1) & 1);
        look_up();
        to_load--;
      }
      f32x4 s[NB];
      if (scores) {
        const lds_u8* t = (lds_u8*)lat[n & 1] + krow * R * 2;
        const lds_u8* u = (lds_u8*)rot[n & 1] + krow * 128;
        const int k0 = fresh((g ^ kf) * 16);
        f32x4 s0[NB] = {}, s1[NB] = {};
#pragma unroll
        for (int k = 0; k < R / 32; k += 2)  // chunk (4 k + g) ^ kf, a constant and two bits away from g ^ kf
#pragma unroll
          for (int b = 0; b < NB; b++) {
            s0[b] = mma32<DT>(lds_read16(t + b * 32 * R + (k0 ^ k % 4 * 64) + k / 4 * 256), q[k], s0[b]);
            s1[b] = mma32<DT>(lds_read16(t + b * 32 * R + (k0 ^ (k + 1) % 4 * 64) + k / 4 * 256), q[k + 1], s1[b]);
          }
#pragma unroll
        for (int k = 0; k < P / 32; k++)
#pragma unroll
          for (int b = 0; b < NB; b++) s0[b] = mma32<DT>(lds_read16(u + b * 16 * 128 + ((4 * k + g) ^ rf) * 16), q[R / 32 + k], s0[b]);
#pragma unroll
        for (int b = 0; b < NB; b++) {
          const float4 v = *(const float4*)&seen[n & 1][(tb + b) * 16 + 4 * g];
          const float vv[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int i = 0; i < 4; i++) s[b][i] = vv[i] != 0.0f ? (s0[b][i] + s1[b][i]) * to_log2 : -__builtin_huge_valf();
          const float top = max_over_rows(fmaxf(fmaxf(s[b][0], s[b][1]), fmaxf(s[b][2], s[b][3])));
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
        lds_u8* const pw = (lds_u8*)prob + at * (kUnit * 2) + 8 * (g & 1);
#pragma unroll
        for (int b = 0; b < NB; b++) {
          float e[4];
#pragma unroll
          for (int i = 0; i < 4; i++) e[i] = __builtin_amdgcn_exp2f(s[b][i] - base);
          l += (e[0] + e[1]) + (e[2] + e[3]);
          // rounded for the matrix cores; the sum l takes them unrounded
          lds_write8(pw + ((2 * (tb + b) + (g >> 1)) ^ pf) * 16, pack2<DT>(e[0], e[1]), pack2<DT>(e[2], e[3]));
        }
      }
      __syncthreads();
      {
        // chunk ch ^ vf of column block c, ch = 2 (wave CB + c) + (col % 4) / 2
        lds_u8* t = (lds_u8*)lat[n & 1] + vrow * R * 2 + 8 * (col & 1) + wave * 2 * CB / 16 * 256;
        const int v0 = fresh(((wave * 2 * CB % 16 + ((col & 3) >> 1)) ^ vf) * 16);
        float f[HB];
        bool changed = false;
#pragma unroll
        for (int h = 0; h < HB; h++) {
          f[h] = fade[h * 16 + col];
          changed |= f[h] != 1.0f;
        }
        if (__any(changed)) {
#pragma unroll
          for (int h = 0; h < HB; h++)
#pragma unroll
            for (int c = 0; c < CB; c++) o[h][c] *= f[h];
        }
#pragma unroll
        for (int k = 0; k < kUnit / 32; k++) {
          s16x8 pb[HB];
#pragma unroll
          for (int h = 0; h < HB; h++) pb[h] = lds_read16((lds_u8*)prob + (h * 16 + col) * (kUnit * 2) + ((4 * k + g) ^ pf) * 16);
#pragma unroll
          for (int c = 0; c < CB; c++) {
            const s16x8 av = join(lds_read_tr(t + k * 64 * R + (v0 ^ 32 * c)), lds_read_tr(t + k * 64 * R + 8 * R + (v0 ^ 32 * c ^ 16)));
#pragma unroll
            for (int h = 0; h < HB; h++) o[h][c] = mma32<DT>(av, pb[h], o[h][c]);
          }
        }
      }
      if (i == units) break;
    }
    n++;
    if (left > 0) {
      do next++;
      while (ld_const(&d.w.items[next].len) == 0);
      load_q(next);
    }

    // the heads' sums of probabilities, over a wave's lanes and the waves of a head block
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (scores && g == 0) {
      tops[HB == 4 ? tb >> 1 : tb][hb * 16 + col] = l;
      if (tb == 0) last_top[hb * 16 + col] = m;
    }
    VIB3_WAIT_VM(0);  // the next queries, before the stores below: those are not waited for
    __syncthreads();
    const bool whole = unit == 0 && units == (len + kUnit - 1) / kUnit;
    const int r = x / groups, h0 = (x - r * groups) * 64;
    const int fcol = fresh(col), fg = fresh(g);
#pragma unroll
    for (int h = 0; h < HB; h++) {
      const int at = h * 16 + fcol, head = h0 + at;
      const float sum = HB == 4 ? tops[0][at] + tops[1][at] : (tops[0][at] + tops[1][at]) + (tops[2][at] + tops[3][at]);
      if (head >= a.heads) continue;
      const int c0 = wave * CB * 16 + 4 * fg;
      if (whole) {
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
        uint16_t* out = d.w.ol + ((size_t)r * a.heads + head) * R + c0;
#pragma unroll
        for (int c = 0; c < CB; c++)
          *(uint2*)(out + 16 * c) =
              make_uint2(pack2<DT>(o[h][c][0] * inv, o[h][c][1] * inv), pack2<DT>(o[h][c][2] * inv, o[h][c][3] * inv));
      } else {
        const size_t slot = (2 * (size_t)blockIdx.x + (first_of_share == 0 ? 0 : 1)) * group_heads(a.heads) + at;
        float* out = d.w.part + slot * R + c0;
#pragma unroll
        for (int c = 0; c < CB; c++) *(float4*)(out + 16 * c) = make_float4(o[h][c][0], o[h][c][1], o[h][c][2], o[h][c][3]);
        if (fg == 0 && wave == 0) d.w.stat[slot] = make_float2(last_top[at], sum);
      }
    }
    if (left == 0) break;
    x = next;
    unit = 0;
    len = ld_const(&d.w.items[x].len);
    units = (int)min((int64_t)((len + kUnit - 1) / kUnit), left);
  }
}

// ------------------------------------------------------------------------- joined rows and W_uv

// A workgroup takes up to 16 rows of one head. Its 16 waves are dealt over the rows: a wave, or where there are fewer rows
// several, joins a row's parts (the weights of all parts first, then the parts' sums, several loads in flight). The rows' weighted latents
// go to LDS in 16 bits, and v_dim / 16 waves multiply them by 16 rows of W_uv each, which they have loaded before the join. Without W_uv the weighted latents are the result.
template <int DT, int R>
__global__ __launch_bounds__(1024) void k_mla_finish(DecodeArgs d) {
  const vib3_mla_decode& a = d.a;
  constexpr int kStride = R + 8;  // 16 bytes more: rows start in different banks
  constexpr int kCols = R / 64;   // columns of a lane
  __shared__ __align__(16) uint16_t lat[16 * kStride];
  __shared__ __align__(16) float sums[16][R];
  const int h = (int)blockIdx.x, r0 = (int)blockIdx.y * 16;
  const int tid = (int)threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, col = lane & 15;
  const int rows = min(16, a.rows - r0);
  const uint16_t* wv = (const uint16_t*)a.kv_b + ((size_t)h * (a.nope + a.v_dim) + a.nope + col) * R + 8 * g;
  s16x8 first[R / 32];
  const bool product = a.kv_b && wave * 16 < a.v_dim;
  if (product) {
#pragma unroll
    for (int k = 0; k < R / 32; k++) first[k] = *(const s16x8*)(wv + (size_t)wave * 16 * R + k * 32);
  }
  const int teams = rows > 8 ? 16 : rows > 4 ? 8 : rows > 2 ? 4 : rows;  // rows joined at a time
  const int per_row = 16 / teams, i = wave / per_row, mate = wave % per_row;
  {
    const int r = r0 + i, x = r * head_groups(a.heads) + h / 64;
    float o[kCols] = {};
    const int64_t per = d.w.head[0];
    const int64_t lo = i < rows ? d.w.items[x].begin : 0, hi = i < rows ? d.w.items[x + 1].begin : 0;
    if (hi > lo) {
      const int w0 = (int)(lo / per), parts = (int)((hi - 1) / per) - w0 + 1;
      if (parts == 1) {
        if (mate == 0) {
          const uint16_t* p = d.w.ol + ((size_t)r * a.heads + h) * R + lane * kCols;
#pragma unroll
          for (int c = 0; c < kCols; c++) o[c] = to_f32<DT>(p[c]);
        }
      } else {
        // part j: slot 2 (w0 + j), but the first one 2 w0 + 1 where its share began with another item
        const bool late = lo != w0 * per;
        const int hg = group_heads(a.heads), hh = h % 64;
        auto place = [&](int j) { return ((size_t)2 * (w0 + j) + (j == 0 && late ? 1 : 0)) * hg + hh; };
        float2 st[kShares / 64];  // lane l: parts l, l + 64, ...
        float m = -__builtin_huge_valf();
#pragma unroll
        for (int k = 0; k < kShares / 64; k++) {
          st[k] = lane + 64 * k < parts ? d.w.stat[place(lane + 64 * k)] : make_float2(-__builtin_huge_valf(), 0.0f);
          m = fmaxf(m, st[k].x);
        }
#pragma unroll
        for (int s = 1; s < 64; s *= 2) m = fmaxf(m, __shfl_xor(m, s));
        const float base = m == -__builtin_huge_valf() ? 0.0f : m;
        float l = 0.0f;
#pragma unroll
        for (int k = 0; k < kShares / 64; k++) {
          st[k].x = __builtin_amdgcn_exp2f(st[k].x - base);
          l += st[k].x * st[k].y;
        }
        l = wave_sum(l);
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
        for (int k = 0; k < kShares / 64; k++) {
#pragma unroll 4
          for (int j = 64 * k + mate; j < min(parts, 64 * k + 64); j += per_row) {
            const float f = __shfl(st[k].x, j - 64 * k) * inv;
            const float* p = d.w.part + place(j) * R + lane * kCols;
#pragma unroll
            for (int c = 0; c < kCols; c += 4) {
              const float4 v = *(const float4*)(p + c);
              o[c] += f * v.x;
              o[c + 1] += f * v.y;
              o[c + 2] += f * v.z;
              o[c + 3] += f * v.w;
            }
          }
        }
      }
    }
#pragma unroll
    for (int c = 0; c < kCols; c += 4) *(float4*)&sums[wave][lane * kCols + c] = make_float4(o[c], o[c + 1], o[c + 2], o[c + 3]);
  }
  __syncthreads();
  for (int at = tid; at < rows * R; at += 1024) {
    const int k = at / R, c = at % R;
    float v = 0.0f;
    for (int s = 0; s < per_row; s++) v += sums[k * per_row + s][c];
    if (a.kv_b) lat[k * kStride + c] = from_f32<DT>(v);
    else ((uint16_t*)a.out)[(int64_t)(r0 + k) * a.out_row_stride + (int64_t)h * a.out_head_stride + c] = from_f32<DT>(v);
  }
  if (!a.kv_b) return;
  __syncthreads();
  if (!product) return;
  const int row = min(col, rows - 1);
  f32x4 acc = {};
#pragma unroll
  for (int k = 0; k < R / 32; k++)  // rows of W_uv times the rows' latents: a lane ends with 4 outputs of one row
    acc = mma32<DT>(first[k], *(const s16x8*)(lat + row * kStride + k * 32 + 8 * g), acc);
  if (col < rows)
    *(uint2*)((uint16_t*)a.out + (int64_t)(r0 + col) * a.out_row_stride + (int64_t)h * a.out_head_stride + wave * 16 + 4 * g) =
        make_uint2(pack2<DT>(acc[0], acc[1]), pack2<DT>(acc[2], acc[3]));
}

template <int DT, int R, int P>
int launch_decode(const DecodeArgs& d, hipStream_t st) {
  const vib3_mla_decode& a = d.a;
  if (a.kv_b) {
    const int col_blocks = R / kAbsorbCols;
    hipLaunchKernelGGL(k_mla_absorb<DT>, dim3((unsigned)(a.heads * col_blocks + 1), (unsigned)((a.rows + kAbsorbRows - 1) / kAbsorbRows)), dim3(256), 0, st,
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
  hipLaunchKernelGGL((k_mla_finish<DT, R>), dim3((unsigned)a.heads, (unsigned)((a.rows + 15) / 16)), dim3(1024), 0, st, d);
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
